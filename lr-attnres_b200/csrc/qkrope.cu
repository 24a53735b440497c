// Per-head RMS norm of queries and keys with the rotation by position, and the
// split of the fused q/k/v projection into heads, in one pass over its rows.
//
//   xhat = x * rsqrt(mean(x^2) + eps)            (normalize; else xhat = x)
//   y    = R(p) (w * xhat)                       w: learned weight, or 1
// R(p) turns the pairs of the first rotary_dim elements -- (2i, 2i+1), or
// (i, i + rotary_dim/2) -- by the angle whose cosine and sine stand in row p of
// two tables; the other elements pass. Value heads are copied. Backward, from x
// and the three gradients:
//   g  = R(p)^T dy,   dw = sum g * xhat,   e = w * g
//   dx = inv * (e - xhat * mean(e * xhat))
// All arithmetic is fp32, each output rounded once. The inverse rms is formed
// again in the backward: x is read there anyway, so nothing is saved.
//
// Bound by HBM: forward 2, backward (with x of q and k read again) 2 2/3 times
// the projection's bytes when query and key heads are as many.
#include <algorithm>

#include "common.cuh"
#include "launch_cache.h"
#include "qkrope.h"

namespace attnres {

// The row of the tables for token n, or -1 when the caller's position lies
// outside them (its q and k rows become NaN rather than reading past the end).
__device__ __forceinline__ long long rope_position(const QkRopeArgs& a, long long n) {
  long long p;
  if (a.positions == nullptr) p = n % a.T;
  else if (a.positions64) p = static_cast<const long long*>(a.positions)[n];
  else p = static_cast<const int*>(a.positions)[n];
  return (p >= 0 && p < a.table_rows) ? p : -1;
}

__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7fffffff); }

// Which of q / k / v head r of a token is, and its index there.
struct HeadRef {
  int part, h;  // part 0 q, 1 k, 2 v
};
__device__ __forceinline__ HeadRef head_ref(const QkRopeArgs& a, int r) {
  if (r < a.Hq) return {0, r};
  if (r < a.Hq + a.Hkv) return {1, r - a.Hq};
  return {2, r - a.Hq - a.Hkv};
}
template <typename T>
__device__ __forceinline__ const T* grad_row(const QkRopeArgs& a, long long n, HeadRef h) {
  return static_cast<const T*>(a.g[h.part]) + (n / a.T) * a.gs[h.part][0] + (n % a.T) * a.gs[h.part][1] +
         h.h * a.gs[h.part][2];
}
template <typename T>
__device__ __forceinline__ T* out_row(const QkRopeArgs& a, long long n, HeadRef h) {
  return static_cast<T*>(a.out[h.part]) + (n * (h.part == 0 ? a.Hq : a.Hkv) + h.h) * a.D;
}

// ---------------------------------------------------------------------------
// any head size, alignment and stride: one warp per (token, head) row, staged
// in shared memory as fp32
// ---------------------------------------------------------------------------
constexpr int kRopeWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kRopeWarps * 32) qkrope_fwd_any_kernel(const __grid_constant__ QkRopeArgs a) {
  extern __shared__ float rope_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* buf = rope_smem + warp * a.D;
  const int H = a.Hq + 2 * a.Hkv;
  const long long row = static_cast<long long>(blockIdx.x) * kRopeWarps + warp;
  if (row >= a.N * H) return;
  const long long n = row / H;
  const int r = static_cast<int>(row % H);
  const HeadRef hr = head_ref(a, r);
  const T* x = static_cast<const T*>(a.qkv) + n * a.qkv_stride + static_cast<long long>(r) * a.D;
  T* y = out_row<T>(a, n, hr);
  if (hr.part == 2) {
    for (int j = lane; j < a.D; j += 32) y[j] = x[j];
    return;
  }
  const T* w = static_cast<const T*>(a.w[hr.part]);
  float ss = 0.f;
  for (int j = lane; j < a.D; j += 32) {
    const float v = Elem<T>::to_f(x[j]);
    ss = fmaf(v, v, ss);
    buf[j] = v;
  }
  ss = warp_sum(ss);
  const float inv = a.normalize ? rsqrtf(ss / a.D + a.eps) : 1.f;
  __syncwarp();
  const long long p = rope_position(a, n);
  const int half = a.rot / 2;
  for (int i = lane; i < half; i += 32) {
    const int i0 = a.interleaved ? 2 * i : i, i1 = a.interleaved ? 2 * i + 1 : i + half;
    float u = buf[i0] * inv, v = buf[i1] * inv;
    if (w) {
      u *= Elem<T>::to_f(w[i0]);
      v *= Elem<T>::to_f(w[i1]);
    }
    const float c = p < 0 ? quiet_nan() : a.cos[p * half + i], s = p < 0 ? quiet_nan() : a.sin[p * half + i];
    y[i0] = Elem<T>::from_f(u * c - v * s);
    y[i1] = Elem<T>::from_f(u * s + v * c);
  }
  for (int j = a.rot + lane; j < a.D; j += 32) {
    const float u = buf[j] * inv;
    y[j] = Elem<T>::from_f(w ? u * Elem<T>::to_f(w[j]) : u);
  }
}

// Weight gradients: each warp sums its rows into its own shared arrays, the
// block adds its warps in order, and rope_weight_sum_kernel the blocks.
template <typename T>
__global__ void __launch_bounds__(kRopeWarps * 32) qkrope_bwd_any_kernel(const __grid_constant__ QkRopeArgs a) {
  extern __shared__ float rope_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = a.D, H = a.Hq + 2 * a.Hkv;
  float* xb = rope_smem + warp * 2 * D;
  float* gb = xb + D;
  float* acc = rope_smem + kRopeWarps * 2 * D + warp * 2 * D;  // [2][D], only with weights
  const bool weighted = a.partials != nullptr;
  if (weighted)
    for (int j = lane; j < 2 * D; j += 32) acc[j] = 0.f;
  const int half = a.rot / 2;
  const long long step = static_cast<long long>(gridDim.x) * kRopeWarps;
  for (long long row = static_cast<long long>(blockIdx.x) * kRopeWarps + warp; row < a.N * H; row += step) {
    const long long n = row / H;
    const int r = static_cast<int>(row % H);
    const HeadRef hr = head_ref(a, r);
    const T* g = grad_row<T>(a, n, hr);
    T* dx = static_cast<T*>(a.dqkv) + (n * H + r) * D;
    if (hr.part == 2) {
      for (int j = lane; j < D; j += 32) dx[j] = g[j];
      continue;
    }
    const T* x = static_cast<const T*>(a.qkv) + n * a.qkv_stride + static_cast<long long>(r) * D;
    const T* w = static_cast<const T*>(a.w[hr.part]);
    __syncwarp();
    float ss = 0.f;
    for (int j = lane; j < D; j += 32) {
      const float v = Elem<T>::to_f(x[j]);
      ss = fmaf(v, v, ss);
      xb[j] = v;
    }
    ss = warp_sum(ss);
    const float inv = a.normalize ? rsqrtf(ss / D + a.eps) : 1.f;
    const long long p = rope_position(a, n);
    for (int i = lane; i < half; i += 32) {
      const int i0 = a.interleaved ? 2 * i : i, i1 = a.interleaved ? 2 * i + 1 : i + half;
      const float u = Elem<T>::to_f(g[i0]), v = Elem<T>::to_f(g[i1]);
      const float c = p < 0 ? quiet_nan() : a.cos[p * half + i], s = p < 0 ? quiet_nan() : a.sin[p * half + i];
      gb[i0] = u * c + v * s;
      gb[i1] = v * c - u * s;
    }
    for (int j = a.rot + lane; j < D; j += 32) gb[j] = Elem<T>::to_f(g[j]);
    __syncwarp();
    float dot = 0.f;
    for (int j = lane; j < D; j += 32) {
      const float xh = xb[j] * inv;
      float e = gb[j];
      if (weighted) acc[hr.part * D + j] += e * xh;
      if (w) e *= Elem<T>::to_f(w[j]);
      gb[j] = e;
      dot = fmaf(e, xh, dot);
    }
    dot = a.normalize ? warp_sum(dot) / D : 0.f;
    for (int j = lane; j < D; j += 32) dx[j] = Elem<T>::from_f(inv * (gb[j] - xb[j] * inv * dot));
  }
  if (!weighted) return;
  __syncthreads();
  for (int j = threadIdx.x; j < 2 * D; j += kRopeWarps * 32) {
    float s = 0.f;
    for (int w = 0; w < kRopeWarps; ++w) s += rope_smem[kRopeWarps * 2 * D + w * 2 * D + j];
    a.partials[static_cast<long long>(blockIdx.x) * 2 * D + j] = s;
  }
}

// dw[j] = sum over the blocks' partials in a fixed order: one warp per column,
// lane l adds blocks l, l + 32, ..., then a butterfly.
template <typename T>
__global__ void __launch_bounds__(128) rope_weight_sum_kernel(const float* __restrict__ partials, int blocks, int D,
                                                              T* __restrict__ dwq, T* __restrict__ dwk) {
  const int col = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (col >= 2 * D) return;
  float s = 0.f;
  for (int b = lane; b < blocks; b += 32) s += partials[static_cast<long long>(b) * 2 * D + col];
  s = warp_sum(s);
  T* out = col < D ? dwq : dwk;
  if (lane == 0 && out) out[col < D ? col : col - D] = Elem<T>::from_f(s);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
namespace {

constexpr int kRopePartialBlocksPerSm = 4;

template <typename T>
cudaError_t forward_t(const QkRopeArgs& a, cudaStream_t st) {
  const long long rows = a.N * (a.Hq + 2 * a.Hkv);
  const long long blocks = (rows + kRopeWarps - 1) / kRopeWarps;
  qkrope_fwd_any_kernel<T><<<static_cast<unsigned>(blocks), kRopeWarps * 32, kRopeWarps * a.D * sizeof(float), st>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t backward_t(const QkRopeArgs& a, cudaStream_t st) {
  int nsm = 0;
  cudaError_t e = cached_sm_count(&nsm);
  if (e != cudaSuccess) return e;
  const long long rows = a.N * (a.Hq + 2 * a.Hkv);
  long long blocks = (rows + kRopeWarps - 1) / kRopeWarps;
  if (a.partials) blocks = std::min<long long>(blocks, static_cast<long long>(nsm) * kRopePartialBlocksPerSm);
  const size_t smem = kRopeWarps * 2 * a.D * sizeof(float) * (a.partials ? 2 : 1);
  qkrope_bwd_any_kernel<T><<<static_cast<unsigned>(blocks), kRopeWarps * 32, smem, st>>>(a);
  if ((e = cudaGetLastError()) != cudaSuccess || !a.partials) return e;
  rope_weight_sum_kernel<T><<<(2 * a.D + 3) / 4, 128, 0, st>>>(a.partials, static_cast<int>(blocks), a.D,
                                                             static_cast<T*>(a.dw[0]), static_cast<T*>(a.dw[1]));
  return cudaGetLastError();
}

}  // namespace

size_t qkrope_workspace_bytes(int D) {
  int nsm = 0;
  if (cached_sm_count(&nsm) != cudaSuccess) nsm = 256;  // no device here: more than any has
  return static_cast<size_t>(nsm) * kRopePartialBlocksPerSm * 2 * D * sizeof(float);
}

cudaError_t qkrope_launch(bool backward, int dtype, const QkRopeArgs& a, cudaStream_t st) {
  switch (dtype) {
    case ATTNRES_DTYPE_F32: return backward ? backward_t<float>(a, st) : forward_t<float>(a, st);
    case ATTNRES_DTYPE_F16: return backward ? backward_t<__half>(a, st) : forward_t<__half>(a, st);
    default: return backward ? backward_t<__nv_bfloat16>(a, st) : forward_t<__nv_bfloat16>(a, st);
  }
}

}  // namespace attnres
