// Writing keys and values into the 4-bit paged cache and reading them back (format:
// kv4.h). For a group of 32 elements x:
//   step = f16((max - min) / 15), low = f16(min)
//   code = clamp(rint((x - low) / step), 0, 15), 0 where step is 0
// with the rounded step and low, so the code is the nearest of the 16 values that will
// be read back. A group that holds an infinity or a NaN gets NaN for step and low and
// reads back as NaN.
//
// Four lanes share a group (8 elements each, two shuffles for its extremes), and a
// thread does the same part of a key and of its value, so that both loads are in
// flight. Bound by HBM and close behind it by issue slots: the quotient is formed with
// the reciprocal and redone by division only within 2^-16 of a tie, which keeps the
// codes those of the division.
#include "common.cuh"
#include "kv4.h"
#include "tma.cuh"

namespace attnres {

static __device__ unsigned int g_kv4_status = 0;

// Row of the pool of token t of sequence b for head 0 (head h is h * page rows on),
// -1 if the token takes no part, -2 if the page table has no page for it.
__device__ __forceinline__ long long kv4_row(const Kv4RowsArgs& a, int b, int t) {
  if (a.counts && t >= a.counts[b]) return -1;
  const long long at = static_cast<long long>(a.start[b]) + t;
  if (at < 0) return -2;
  const long long slot = at / a.c.page;
  if (slot >= a.max_pages) return -2;
  const int page = a.table[b * a.table_stride + slot];
  if (page < 0 || page >= a.c.pages) return -2;
  return static_cast<long long>(page) * a.c.heads * a.c.page + (at - slot * a.c.page);
}

// 8 consecutive elements as fp32, by 16-byte loads where the row allows.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool packs, float (&x)[8]) {
  if (packs) {
    constexpr int VEC = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += VEC) {
      const Pack<T, VEC> v = load_stream<T, VEC>(p + i);
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[i + e] = Elem<T>::to_f(v.e[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = Elem<T>::to_f(p[e]);
  }
}

struct Quantised {
  uint32_t codes;  // element e in bits 4e .. 4e + 3
  __half2 params;  // step, low
};

// The four lanes of a group call this together.
__device__ __forceinline__ Quantised quantise8(const float (&x)[8]) {
  float top = x[0], low = x[0];
  bool odd = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    top = fmaxf(top, x[e]);
    low = fminf(low, x[e]);
    odd |= !(fabsf(x[e]) <= 3.402823466e38f);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    odd |= __shfl_xor_sync(0xffffffffu, static_cast<int>(odd), o) != 0;
  }
  Quantised r;
  const float nan = __int_as_float(0x7fffffff);
  r.params = odd ? __floats2half2_rn(nan, nan)
                 : __floats2half2_rn(__fmul_rn(__fsub_rn(top, low), 1.f / 15.f), low);
  const float step = __low2float(r.params), base = __high2float(r.params);
  r.codes = 0;
  if (step > 0.f) {
    const float inv = __frcp_rn(step);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = __fsub_rn(x[e], base), quotient = d * inv;
      float n = rintf(quotient);
      if (fabsf(quotient - n) > 0.5f - 1.f / 65536.f) n = rintf(__fdiv_rn(d, step));
      r.codes |= static_cast<uint32_t>(fminf(fmaxf(n, 0.f), 15.f)) << (4 * e);
    }
  }
  return r;
}

template <typename T>
__global__ void __launch_bounds__(256) kv4_append_kernel(const __grid_constant__ Kv4RowsArgs a, bool packs) {
  const int G = a.c.D / kKv4Group;
  const long long quad = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 2;
  const int c = threadIdx.x & 3;
  const long long total = static_cast<long long>(a.B) * a.T * a.c.heads * G;
  const bool live = quad < total;  // whole groups; the shuffles need every lane
  long long i = live ? quad : 0;
  const int g = static_cast<int>(i % G);
  i /= G;
  const int h = static_cast<int>(i % a.c.heads);
  i /= a.c.heads;
  const int t = static_cast<int>(i % a.T), b = static_cast<int>(i / a.T);
  const long long base = live ? kv4_row(a, b, t) : -1;
  float k[8] = {}, v[8] = {};
  if (base >= 0) {
    const int e = g * kKv4Group + c * 8;
    load8<T>(static_cast<const T*>(a.k) + b * a.ks[0] + t * a.ks[1] + h * a.ks[2] + e, packs, k);
    load8<T>(static_cast<const T*>(a.v) + b * a.vs[0] + t * a.vs[1] + h * a.vs[2] + e, packs, v);
  }
  const Quantised qk = quantise8(k), qv = quantise8(v);
  if (base < 0) {
    if (base == -2) atomicOr(&g_kv4_status, kStatusCacheRange);
    return;
  }
  const long long row = base + static_cast<long long>(h) * a.c.page;
  reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(a.c.k_codes) + row * (a.c.D / 2))[c * G + g] = qk.codes;
  uint16_t* vc = reinterpret_cast<uint16_t*>(static_cast<unsigned char*>(a.c.v_codes) + row * (a.c.D / 2));
  vc[2 * c * G + g] = static_cast<uint16_t>(qv.codes);
  vc[(2 * c + 1) * G + g] = static_cast<uint16_t>(qv.codes >> 16);
  if (c == 0) static_cast<__half2*>(a.c.k_params)[row * G + g] = qk.params;
  if (c == 1) static_cast<__half2*>(a.c.v_params)[row * G + g] = qv.params;
}

template <typename T>
__device__ __forceinline__ void store_values(T* out, uint32_t codes, __half2 params, bool there) {
  const float step = __low2float(params), low = __high2float(params);
  constexpr int VEC = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8; i += VEC) {
    float y[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      y[e] = there ? __fadd_rn(low, __fmul_rn(step, static_cast<float>((codes >> (4 * (i + e))) & 15u))) : 0.f;
    store_pack<T, VEC>(out + i, y);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ Kv4RowsArgs a) {
  const int G = a.c.D / kKv4Group;
  const long long quad = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 2;
  const int c = threadIdx.x & 3;
  if (quad >= static_cast<long long>(a.B) * a.T * a.c.heads * G) return;
  long long i = quad;
  const int g = static_cast<int>(i % G);
  i /= G;
  const int h = static_cast<int>(i % a.c.heads);
  i /= a.c.heads;
  const int t = static_cast<int>(i % a.T), b = static_cast<int>(i / a.T);
  const long long base = kv4_row(a, b, t);
  uint32_t kw = 0, vw = 0;
  __half2 kp = __half2{}, vp = __half2{};
  if (base >= 0) {
    const long long row = base + static_cast<long long>(h) * a.c.page;
    kw = reinterpret_cast<const uint32_t*>(static_cast<const unsigned char*>(a.c.k_codes) + row * (a.c.D / 2))[c * G + g];
    const uint16_t* vc = reinterpret_cast<const uint16_t*>(static_cast<const unsigned char*>(a.c.v_codes) + row * (a.c.D / 2));
    vw = vc[2 * c * G + g] | (static_cast<uint32_t>(vc[(2 * c + 1) * G + g]) << 16);
    kp = static_cast<const __half2*>(a.c.k_params)[row * G + g];
    vp = static_cast<const __half2*>(a.c.v_params)[row * G + g];
  } else if (base == -2) {
    atomicOr(&g_kv4_status, kStatusCacheRange);
  }
  const long long to = quad * kKv4Group + c * 8;
  store_values<T>(static_cast<T*>(a.k_out) + to, kw, kp, base >= 0);
  store_values<T>(static_cast<T*>(a.v_out) + to, vw, vp, base >= 0);
}

namespace {

unsigned blocks_of(const Kv4RowsArgs& a) {
  const long long threads = 4LL * a.B * a.T * a.c.heads * (a.c.D / kKv4Group);
  return static_cast<unsigned>((threads + 255) / 256);
}

template <typename T>
cudaError_t append_t(const Kv4RowsArgs& a, cudaStream_t st) {
  bool packs = (reinterpret_cast<uintptr_t>(a.k) & 15u) == 0 && (reinterpret_cast<uintptr_t>(a.v) & 15u) == 0;
  for (int i = 0; i < 3; ++i) packs = packs && a.ks[i] * sizeof(T) % 16 == 0 && a.vs[i] * sizeof(T) % 16 == 0;
  kv4_append_kernel<T><<<blocks_of(a), 256, 0, st>>>(a, packs);
  return cudaGetLastError();
}

}  // namespace

cudaError_t kv4_append_launch(int dtype, const Kv4RowsArgs& a, cudaStream_t st) {
  switch (dtype) {
    case ATTNRES_DTYPE_F32: return append_t<float>(a, st);
    case ATTNRES_DTYPE_F16: return append_t<__half>(a, st);
    default: return append_t<__nv_bfloat16>(a, st);
  }
}

cudaError_t kv4_read_launch(int dtype, const Kv4RowsArgs& a, cudaStream_t st) {
  const unsigned grid = blocks_of(a);
  switch (dtype) {
    case ATTNRES_DTYPE_F32: kv4_read_kernel<float><<<grid, 256, 0, st>>>(a); break;
    case ATTNRES_DTYPE_F16: kv4_read_kernel<__half><<<grid, 256, 0, st>>>(a); break;
    default: kv4_read_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
  }
  return cudaGetLastError();
}

cudaError_t read_kv4_status(unsigned* status, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_kv4_status, sizeof(unsigned));
  if (e != cudaSuccess || !reset) return e;
  const unsigned zero = 0;
  return cudaMemcpyToSymbol(g_kv4_status, &zero, sizeof(unsigned));
}

}  // namespace attnres
