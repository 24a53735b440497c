// Launch bundle of the gated projection (swiglu.cu).
#pragma once

#include <cuda_runtime.h>

namespace attnres {

struct SwigluArgs {
  long long N;
  int C, F;
  const void *x, *w;  // [N, C], [2F, C] (value rows, then gate rows)
  long long x_stride, w_stride;
  void* out;  // forward: h [N, F]
  // backward
  const void* dh;  // [N, F]
  long long dh_stride;
  void *dx, *dw;    // [N, C], [2F, C], either may be null
  void* workspace;  // [N, 2F] of the data's type: du | dg
};

cudaError_t swiglu_launch(bool backward, int dtype, const SwigluArgs& s, cudaStream_t st);
cudaError_t read_swiglu_status(unsigned* status, bool reset);

}  // namespace attnres
