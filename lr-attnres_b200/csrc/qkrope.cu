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
// the projection's bytes when query and key heads are as many. 16384 tokens of 16
// query and key heads of 64, bf16: forward 34.4 us for 201 MB (5.9 TB/s, 91 % of the
// measured copy rate), backward 56.8 us for 277 MB (4.9 TB/s, 76 %).
#include <algorithm>

#include "common.cuh"
#include "launch_cache.h"
#include "qkrope.h"

namespace attnres {

// The row of the tables for token n, or -1 when the caller's position lies
// outside them (its q and k rows become NaN rather than reading past the end).
__device__ __forceinline__ long long rope_position(const QkRopeArgs& a, long long n, long long t) {
  long long p;
  if (a.positions == nullptr) p = t;
  else if (a.positions64) p = static_cast<const long long*>(a.positions)[n];
  else p = static_cast<const int*>(a.positions)[n];
  return (p >= 0 && p < a.table_rows) ? p : -1;
}

// Element j of the norm weight of the queries (0) or keys (1): fp32 weights multiply as they
// are, and their gradients are not rounded to the data's type either.
template <typename T>
__device__ __forceinline__ float rope_weight(const QkRopeArgs& a, int part, int j) {
  return a.w32 ? static_cast<const float*>(a.w[part])[j] : Elem<T>::to_f(static_cast<const T*>(a.w[part])[j]);
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
__device__ __forceinline__ const T* grad_row(const QkRopeArgs& a, long long b, long long t, HeadRef h) {
  return static_cast<const T*>(a.g[h.part]) + b * a.gs[h.part][0] + t * a.gs[h.part][1] + h.h * a.gs[h.part][2];
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
  const bool w = a.w[hr.part] != nullptr;
  float ss = 0.f;
  for (int j = lane; j < a.D; j += 32) {
    const float v = Elem<T>::to_f(x[j]);
    ss = fmaf(v, v, ss);
    buf[j] = v;
  }
  ss = warp_sum(ss);
  const float inv = a.normalize ? rsqrtf(ss / a.D + a.eps) : 1.f;
  __syncwarp();
  const long long p = rope_position(a, n, n % a.T);
  const int half = a.rot / 2;
  for (int i = lane; i < half; i += 32) {
    const int i0 = a.interleaved ? 2 * i : i, i1 = a.interleaved ? 2 * i + 1 : i + half;
    float u = buf[i0] * inv, v = buf[i1] * inv;
    if (w) {
      u *= rope_weight<T>(a, hr.part, i0);
      v *= rope_weight<T>(a, hr.part, i1);
    }
    const float c = p < 0 ? quiet_nan() : a.cos[p * half + i], s = p < 0 ? quiet_nan() : a.sin[p * half + i];
    y[i0] = Elem<T>::from_f(u * c - v * s);
    y[i1] = Elem<T>::from_f(u * s + v * c);
  }
  for (int j = a.rot + lane; j < a.D; j += 32) {
    const float u = buf[j] * inv;
    y[j] = Elem<T>::from_f(w ? u * rope_weight<T>(a, hr.part, j) : u);
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
    const T* g = grad_row<T>(a, n / a.T, n % a.T, hr);
    T* dx = static_cast<T*>(a.dqkv) + (n * H + r) * D;
    if (hr.part == 2) {
      for (int j = lane; j < D; j += 32) dx[j] = g[j];
      continue;
    }
    const T* x = static_cast<const T*>(a.qkv) + n * a.qkv_stride + static_cast<long long>(r) * D;
    const bool w = a.w[hr.part] != nullptr;
    __syncwarp();
    float ss = 0.f;
    for (int j = lane; j < D; j += 32) {
      const float v = Elem<T>::to_f(x[j]);
      ss = fmaf(v, v, ss);
      xb[j] = v;
    }
    ss = warp_sum(ss);
    const float inv = a.normalize ? rsqrtf(ss / D + a.eps) : 1.f;
    const long long p = rope_position(a, n, n % a.T);
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
      if (w) e *= rope_weight<T>(a, hr.part, j);
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

// ---------------------------------------------------------------------------
// rows of 16-byte packs: a group of G lanes holds a head row, one pack a lane
// ---------------------------------------------------------------------------
// Unit of work of a warp: rope_rounds() rounds of 32 / G consecutive heads of one
// token, so that a round is one contiguous stretch of the projection's row, the
// loads of all rounds are in flight at once and the token's cosines and sines
// are read once per unit. Element pairs: interleaved pairs lie in one lane's
// pack; of half-split pairs lane l < h (h = rotary_dim / 2 / VEC) holds the first
// elements and lane l + h the second, exchanged by a shuffle. Units are counted in
// 32 bits (64-bit divisions took half the backward's time); the host sends
// launches with more of them to the kernels above.
// Rounds of a unit. The weight gradients' sums take registers that four rounds' loads
// need: 1237 x 3 tokens of 20 + 4 heads of 128, backward: 42.7 us with 4, 34.1 with 2
// (without weights 16384 tokens of 16 heads of 64: 60.6 us with 4, 75.6 with 2).
constexpr int rope_rounds(bool backward, bool weighted) { return backward && weighted ? 2 : 4; }
constexpr int kRopeVecThreads = 256;

// Left as single loads, divisions and conversions this was bound by issue slots,
// not by HBM (168 instructions a round, 3.0 TB/s); hence the compile-time pairing,
// packed fp32 arithmetic and one base pointer per part of the row.
template <int VEC> struct RopeLane {
  float c[VEC], s[VEC];  // cosine, and sine with the sign this element's partner takes
  bool turns;
};

// y_j = x_j c_j + partner_j s_j with the sines signed: a' = a c - b s, b' = b c + a s.
// sign = -1 turns backward (the transposed rotation).
template <int VEC, bool INTERLEAVED>
__device__ __forceinline__ RopeLane<VEC> rope_lane(const QkRopeArgs& a, long long p, int l, float sign) {
  RopeLane<VEC> r;
  const int j0 = l * VEC, half = a.rot / 2;
  r.turns = j0 < a.rot;
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    r.c[e] = 1.f;
    r.s[e] = 0.f;
  }
  if (!r.turns) return r;
  if (p < 0) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.c[e] = r.s[e] = quiet_nan();
    return r;
  }
  if constexpr (INTERLEAVED) {
    const Pack<float, VEC / 2> c = load_pack<float, VEC / 2>(a.cos + p * half + j0 / 2);
    const Pack<float, VEC / 2> s = load_pack<float, VEC / 2>(a.sin + p * half + j0 / 2);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      r.c[e] = c.e[e / 2];
      r.s[e] = ((e & 1) ? sign : -sign) * s.e[e / 2];
    }
  } else {
    const bool second = j0 >= half;
    const long long at = p * half + (second ? j0 - half : j0);
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const Pack<float, 4> c = load_pack<float, 4>(a.cos + at + i), s = load_pack<float, 4>(a.sin + at + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        r.c[i + e] = c.e[e];
        r.s[i + e] = (second ? sign : -sign) * s.e[e];
      }
    }
  }
  return r;
}

// Every lane of the warp takes part (the shuffle); lanes that do not turn have
// c = 1, s = 0 and themselves as partner.
template <int VEC, bool INTERLEAVED>
__device__ __forceinline__ void rope_turn(const RopeLane<VEC>& r, int from, float (&x)[VEC]) {
  float partner[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    partner[e] = INTERLEAVED ? x[e ^ 1] : __shfl_sync(0xffffffffu, x[e], from);
  if (INTERLEAVED && !r.turns) return;
#pragma unroll
  for (int e = 0; e < VEC; ++e) x[e] = fmaf(x[e], r.c[e], partner[e] * r.s[e]);
}

__device__ __forceinline__ int rope_partner_lane(const QkRopeArgs& a, bool turns, int l, int vec) {
  const int h = a.rot / 2 / vec, lane = threadIdx.x & 31;
  return !turns ? lane : (l < h ? lane + h : lane - h);
}

template <typename T, int VEC>
__device__ __forceinline__ void widen(const Pack<T, VEC>& x, float (&v)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) unpack2<T, VEC>(x, i, v[2 * i], v[2 * i + 1]);
}

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> narrow(const float (&v)[VEC]) {
  Pack<T, VEC> r;
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.e[e] = v[e];
  } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) reinterpret_cast<__half2*>(r.e)[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i)
      reinterpret_cast<__nv_bfloat162*>(r.e)[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  }
  return r;
}

// The outputs do not displace the rows still to be read from L2 (98 -> 91 us, forward
// and backward of 16384 tokens of 16 heads of 64).
template <typename T, int VEC>
__device__ __forceinline__ void store_streaming(T* p, const Pack<T, VEC>& x) {
  __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&x));
}

template <int VEC>
__device__ __forceinline__ float dot(const float (&x)[VEC], const float (&y)[VEC]) {
  float a0 = 0.f, a1 = 0.f;
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) fma2v(a0, a1, x[2 * i], x[2 * i + 1], y[2 * i], y[2 * i + 1]);
  return a0 + a1;
}
template <int VEC>
__device__ __forceinline__ void scale(float (&x)[VEC], float w) {
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) mul2(x[2 * i], x[2 * i + 1], w, x[2 * i], x[2 * i + 1]);
}

// W: the weights' type, void without weights (as a test at run time the type took registers:
// the half-split forward 19.4 us instead of 17.8 at 1237 x 3 tokens of 20 + 4 heads of 128).
template <typename T, int G, bool INTERLEAVED, typename W>
__global__ void __launch_bounds__(kRopeVecThreads, sizeof(T) == 2 ? 4 : 3)
    qkrope_fwd_kernel(const __grid_constant__ QkRopeArgs a) {
  constexpr bool WEIGHTED = !std::is_void<W>::value;
  constexpr int VEC = 16 / sizeof(T), ROUND = 32 / G, ROUNDS = rope_rounds(false, WEIGHTED);
  const int lane = threadIdx.x & 31, l = lane % G;
  const int H = a.Hq + 2 * a.Hkv, Hqk = a.Hq + a.Hkv;
  const unsigned units = (H + ROUNDS * ROUND - 1) / (ROUNDS * ROUND);
  const unsigned unit = blockIdx.x * (kRopeVecThreads / 32) + (threadIdx.x >> 5);
  if (unit >= static_cast<unsigned>(a.N) * units) return;
  const unsigned n = unit / units;
  const int first = static_cast<int>(unit - n * units) * ROUNDS * ROUND, r0 = first + lane / G;
  const bool mine = l * VEC < a.D;  // lanes beyond the head carry zeros
  const long long p = first < Hqk ? rope_position(a, n, n % static_cast<unsigned>(a.T)) : 0;
  const T* x0 = static_cast<const T*>(a.qkv) + n * a.qkv_stride + l * VEC;
  Pack<T, VEC> x[ROUNDS];
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int r = r0 + i * ROUND;
    if (mine && r < H) x[i] = load_stream<T, VEC>(x0 + r * a.D);
    else x[i] = Pack<T, VEC>{};
  }
  // where head r = 0 of the row would lie in each of the three outputs
  T* const yq = static_cast<T*>(a.out[0]) + static_cast<long long>(n) * a.Hq * a.D + l * VEC;
  T* const yk = static_cast<T*>(a.out[1]) + (static_cast<long long>(n) * a.Hkv - a.Hq) * a.D + l * VEC;
  T* const yv = static_cast<T*>(a.out[2]) + (static_cast<long long>(n) * a.Hkv - Hqk) * a.D + l * VEC;
  RopeLane<VEC> turn;
  float wq[VEC], wk[VEC];
  int from = lane;
  if (first < Hqk) {
    turn = rope_lane<VEC, INTERLEAVED>(a, p, l, 1.f);
    from = rope_partner_lane(a, turn.turns, l, VEC);
    if constexpr (WEIGHTED) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        wq[e] = a.w[0] && mine ? Elem<W>::to_f(static_cast<const W*>(a.w[0])[l * VEC + e]) : 1.f;
        wk[e] = a.w[1] && mine ? Elem<W>::to_f(static_cast<const W*>(a.w[1])[l * VEC + e]) : 1.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int r = r0 + i * ROUND;
    if (first + i * ROUND < Hqk) {  // some head of the round turns (the same for the whole warp)
      float v[VEC];
      widen<T, VEC>(x[i], v);
      if (a.normalize) scale<VEC>(v, rsqrtf(group_sum(dot<VEC>(v, v), G) * a.inv_D + a.eps));
      if (WEIGHTED) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] *= r < a.Hq ? wq[e] : wk[e];
      }
      rope_turn<VEC, INTERLEAVED>(turn, from, v);
      if (r < Hqk) x[i] = narrow<T, VEC>(v);
    }
    if (mine && r < H) store_streaming<T, VEC>((r < a.Hq ? yq : (r < Hqk ? yk : yv)) + r * a.D, x[i]);
  }
}

// WEIGHTED also carries the weight gradients: a lane keeps its columns' sums over
// the units its warp walks through, the block adds its lanes in a fixed order.
template <typename T, int G, bool INTERLEAVED, typename W>
__global__ void __launch_bounds__(kRopeVecThreads, std::is_void<W>::value ? 3 : 2)
    qkrope_bwd_kernel(const __grid_constant__ QkRopeArgs a) {
  constexpr bool WEIGHTED = !std::is_void<W>::value;
  constexpr int VEC = 16 / sizeof(T), ROUND = 32 / G, ROUNDS = rope_rounds(true, WEIGHTED);
  const int lane = threadIdx.x & 31, l = lane % G;
  const int H = a.Hq + 2 * a.Hkv, Hqk = a.Hq + a.Hkv;
  const unsigned units = (H + ROUNDS * ROUND - 1) / (ROUNDS * ROUND);
  const bool mine = l * VEC < a.D;
  float wq[VEC], wk[VEC], acc[2][VEC];
  if constexpr (WEIGHTED) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      wq[e] = a.w[0] && mine ? Elem<W>::to_f(static_cast<const W*>(a.w[0])[l * VEC + e]) : 1.f;
      wk[e] = a.w[1] && mine ? Elem<W>::to_f(static_cast<const W*>(a.w[1])[l * VEC + e]) : 1.f;
      acc[0][e] = acc[1][e] = 0.f;
    }
  }
  const unsigned step = gridDim.x * (kRopeVecThreads / 32), total = static_cast<unsigned>(a.N) * units;
  for (unsigned unit = blockIdx.x * (kRopeVecThreads / 32) + (threadIdx.x >> 5); unit < total; unit += step) {
    const unsigned n = unit / units, b = n / static_cast<unsigned>(a.T), t = n - b * static_cast<unsigned>(a.T);
    const int first = static_cast<int>(unit - n * units) * ROUNDS * ROUND, r0 = first + lane / G;
    const long long p = first < Hqk ? rope_position(a, n, t) : 0;
    const T* x0 = static_cast<const T*>(a.qkv) + n * a.qkv_stride + l * VEC;
    const T* g0[3];
    const int skip[3] = {0, a.Hq, Hqk};
#pragma unroll
    for (int i = 0; i < 3; ++i)
      g0[i] = static_cast<const T*>(a.g[i]) + b * a.gs[i][0] + t * a.gs[i][1] - skip[i] * a.gs[i][2] + l * VEC;
    Pack<T, VEC> x[ROUNDS], g[ROUNDS];
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      const int r = r0 + i * ROUND, part = r < a.Hq ? 0 : (r < Hqk ? 1 : 2);
      x[i] = g[i] = Pack<T, VEC>{};
      if (mine && r < H) {
        g[i] = load_stream<T, VEC>((part == 0 ? g0[0] : (part == 1 ? g0[1] : g0[2])) +
                                   r * (part == 0 ? a.gs[0][2] : (part == 1 ? a.gs[1][2] : a.gs[2][2])));
        if (part < 2) x[i] = load_stream<T, VEC>(x0 + r * a.D);
      }
    }
    RopeLane<VEC> turn;
    int from = lane;
    if (first < Hqk) {
      turn = rope_lane<VEC, INTERLEAVED>(a, p, l, -1.f);
      from = rope_partner_lane(a, turn.turns, l, VEC);
    }
    T* const dx = static_cast<T*>(a.dqkv) + static_cast<long long>(n) * H * a.D + l * VEC;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      const int r = r0 + i * ROUND;
      if (first + i * ROUND < Hqk) {
        float e[VEC], v[VEC];
        widen<T, VEC>(g[i], e);
        widen<T, VEC>(x[i], v);
        rope_turn<VEC, INTERLEAVED>(turn, from, e);
        const float inv = a.normalize ? rsqrtf(group_sum(dot<VEC>(v, v), G) * a.inv_D + a.eps) : 1.f;
        scale<VEC>(v, inv);
        if (WEIGHTED) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            if (r < a.Hq) acc[0][j] = fmaf(e[j], v[j], acc[0][j]);
            else if (r < Hqk) acc[1][j] = fmaf(e[j], v[j], acc[1][j]);
            e[j] *= r < a.Hq ? wq[j] : wk[j];
          }
        }
        const float mean = a.normalize ? group_sum(dot<VEC>(e, v), G) * a.inv_D : 0.f;
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) fma2(e[2 * j], e[2 * j + 1], -mean, v[2 * j], v[2 * j + 1]);
        scale<VEC>(e, inv);
        if (r < Hqk) g[i] = narrow<T, VEC>(e);
      }
      if (mine && r < H) store_streaming<T, VEC>(dx + r * a.D, g[i]);
    }
  }
  if constexpr (WEIGHTED) {
    if (a.partials == nullptr) return;
    extern __shared__ float rope_smem[];  // [kRopeVecThreads][2][VEC]
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) rope_smem[(threadIdx.x * 2 + i) * VEC + j] = acc[i][j];
    __syncthreads();
    for (int col = threadIdx.x; col < 2 * a.D; col += kRopeVecThreads) {
      const int i = col >= a.D, j = col - i * a.D;
      float s = 0.f;
      for (int t = j / VEC; t < kRopeVecThreads; t += G) s += rope_smem[(t * 2 + i) * VEC + j % VEC];
      a.partials[static_cast<long long>(blockIdx.x) * 2 * a.D + col] = s;
    }
  }
}

// dw[j] = sum over the blocks' partials in a fixed order: one warp per column,
// lane l adds blocks l, l + 32, ..., then a butterfly.
template <typename W>
__global__ void __launch_bounds__(128) rope_weight_sum_kernel(const float* __restrict__ partials, int blocks, int D,
                                                              W* __restrict__ dwq, W* __restrict__ dwk) {
  const int col = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (col >= 2 * D) return;
  float s = 0.f;
  for (int b = lane; b < blocks; b += 32) s += partials[static_cast<long long>(b) * 2 * D + col];
  s = warp_sum(s);
  W* out = col < D ? dwq : dwk;
  if (lane == 0 && out) out[col < D ? col : col - D] = Elem<W>::from_f(s);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
namespace {

constexpr int kRopePartialBlocksPerSm = 4;

// Lanes of a head row when it can be moved in 16-byte packs of which each turns
// whole or not at all, else 0: rows and tables 16-byte aligned, at most
// 32 packs a head.
template <typename T>
int pack_lanes(const QkRopeArgs& a, bool backward) {
  constexpr int VEC = 16 / sizeof(T);
  const auto bad = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; };
  if (a.D % VEC || a.D > 32 * VEC || a.qkv_stride % VEC || a.rot % (a.interleaved ? VEC : 2 * VEC)) return 0;
  if (bad(a.qkv) || (a.rot && (bad(a.cos) || bad(a.sin)))) return 0;
  for (int i = 0; i < 3; ++i) {
    if (backward) {
      if (bad(a.g[i])) return 0;
      for (int j = 0; j < 3; ++j)
        if (a.gs[i][j] % VEC) return 0;
    } else if (bad(a.out[i])) {
      return 0;
    }
  }
  if (backward && bad(a.dqkv)) return 0;
  int G = 8;
  while (G * VEC < a.D) G *= 2;
  return a.N * (a.Hq + 2 * a.Hkv) < (1LL << 30) ? G : 0;  // units in 32 bits
}

template <typename T, int G>
cudaError_t vector_t(bool backward, const QkRopeArgs& a, unsigned blocks, cudaStream_t st) {
  using Kernel = void (*)(QkRopeArgs);
  static const Kernel kernels[2][2][3] = {  // without weights, of the data's type, fp32
      {{qkrope_fwd_kernel<T, G, false, void>, qkrope_fwd_kernel<T, G, false, T>, qkrope_fwd_kernel<T, G, false, float>},
       {qkrope_fwd_kernel<T, G, true, void>, qkrope_fwd_kernel<T, G, true, T>, qkrope_fwd_kernel<T, G, true, float>}},
      {{qkrope_bwd_kernel<T, G, false, void>, qkrope_bwd_kernel<T, G, false, T>, qkrope_bwd_kernel<T, G, false, float>},
       {qkrope_bwd_kernel<T, G, true, void>, qkrope_bwd_kernel<T, G, true, T>, qkrope_bwd_kernel<T, G, true, float>}}};
  const size_t smem = a.partials ? kRopeVecThreads * 2 * (16 / sizeof(T)) * sizeof(float) : 0;
  kernels[backward][a.interleaved != 0][a.w[0] || a.w[1] ? 1 + a.w32 : 0]<<<blocks, kRopeVecThreads, smem, st>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t run_t(bool backward, const QkRopeArgs& a, cudaStream_t st) {
  int nsm = 0;
  cudaError_t e = cached_sm_count(&nsm);
  if (e != cudaSuccess) return e;
  const int H = a.Hq + 2 * a.Hkv, G = pack_lanes<T>(a, backward);
  const int warps = G ? kRopeVecThreads / 32 : kRopeWarps;
  const int per_unit = G ? rope_rounds(backward, a.w[0] || a.w[1]) * (32 / G) : 1;
  const long long units = a.N * ((H + per_unit - 1) / per_unit);
  long long blocks = (units + warps - 1) / warps;
  if (a.partials) blocks = std::min<long long>(blocks, static_cast<long long>(nsm) * kRopePartialBlocksPerSm);
  const unsigned grid = static_cast<unsigned>(blocks);
  switch (G) {
    case 8: e = vector_t<T, 8>(backward, a, grid, st); break;
    case 16: e = vector_t<T, 16>(backward, a, grid, st); break;
    case 32: e = vector_t<T, 32>(backward, a, grid, st); break;
    default: {
      const size_t row = kRopeWarps * a.D * sizeof(float);
      if (backward) qkrope_bwd_any_kernel<T><<<grid, kRopeWarps * 32, row * (a.partials ? 4 : 2), st>>>(a);
      else qkrope_fwd_any_kernel<T><<<grid, kRopeWarps * 32, row, st>>>(a);
      e = cudaGetLastError();
    }
  }
  if (e != cudaSuccess || !a.partials) return e;
  const unsigned sums = (2 * a.D + 3) / 4;
  const int n = static_cast<int>(blocks);
  if (a.w32) rope_weight_sum_kernel<<<sums, 128, 0, st>>>(a.partials, n, a.D, static_cast<float*>(a.dw[0]), static_cast<float*>(a.dw[1]));
  else rope_weight_sum_kernel<<<sums, 128, 0, st>>>(a.partials, n, a.D, static_cast<T*>(a.dw[0]), static_cast<T*>(a.dw[1]));
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
    case ATTNRES_DTYPE_F32: return run_t<float>(backward, a, st);
    case ATTNRES_DTYPE_F16: return run_t<__half>(backward, a, st);
    default: return run_t<__nv_bfloat16>(backward, a, st);
  }
}

}  // namespace attnres
