// Writing keys and values into the 4-bit paged cache and reading them back (format:
// kv4.h). For a group of 32 elements x:
//   step = f16((max - min) / 15), low = f16(min)
//   code = clamp(rint((x - low) / step), 0, 15), 0 where step is 0
// with the rounded step and low, so the code is the nearest of the 16 values that will
// be read back. A group that holds an infinity or a NaN, or whose step or low overflows
// float16 (a least value that rounds beyond +-65504, a range of 15 times that), gets NaN for
// step and low and reads back as NaN.
//
// Four lanes share a group (8 elements each, two shuffles for its extremes), and a
// thread does the same part of a key and of its value, of two groups next to each other
// where a head has an even number: four loads in flight, and one look at the page table.
// HBM is the floor, issue slots are what it meets first (a thread has 20 bytes for every
// 16 elements it forms), so the work per element is kept to a subtraction, a
// product, a sum that rounds (adding 1.5 * 2^23 leaves the integer in the low bits), a
// multiply-add into the packed word, and the distance to a tie: the quotient is formed
// with the reciprocal, and elements within 2^-16 of a tie are redone by division, which
// keeps the codes those of the division. 24006 tokens of 8 heads of 128 in bf16, 129 MB
// each way: written in 42 us (3.1 TB/s, three quarters of the issue slots taken), read
// back in 18.9 us (6.8 TB/s; part of the cache is still in L2).
#include "common.cuh"
#include "kv4.h"
#include "tma.cuh"

namespace attnres {

static __device__ unsigned int g_kv4_status = 0;

// Which group of which token a thread's quad of lanes has. Everything is counted in 32
// bits (the host refuses more groups than that): 64-bit divisions were most of the time.
struct GroupRef {
  unsigned g, h, t, b;  // g: the first of N groups
};
template <int N>
__device__ __forceinline__ GroupRef group_ref(const Kv4RowsArgs& a, unsigned quad) {
  const unsigned G = a.c.D / kKv4Group / N;
  GroupRef r;
  unsigned i = quad / G;
  r.g = (quad - i * G) * N;
  const unsigned j = i / a.c.heads;
  r.h = i - j * a.c.heads;
  r.b = j / a.T;
  r.t = j - r.b * a.T;
  return r;
}

// Row of the pool of the group's token and head, -1 if the token takes no part, -2 if the
// page table has no page for it.
__device__ __forceinline__ long long kv4_row(const Kv4RowsArgs& a, const GroupRef& r) {
  if (a.counts && static_cast<int>(r.t) >= a.counts[r.b]) return -1;
  const int start = a.start[r.b];
  const unsigned at = static_cast<unsigned>(start) + r.t;  // below 2^32: both are below 2^31
  if (start < 0) return -2;
  const unsigned slot = at / a.c.page;
  if (slot >= static_cast<unsigned>(a.max_pages)) return -2;
  const int page = a.table[r.b * a.table_stride + slot];
  if (page < 0 || page >= a.c.pages) return -2;
  return (static_cast<long long>(page) * a.c.heads + r.h) * a.c.page + (at - slot * a.c.page);
}

// 8 consecutive elements as fp32, PACKS: by 16-byte loads.
template <typename T, bool PACKS>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (PACKS) {
    constexpr int VEC = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += VEC) {
      const Pack<T, VEC> v = load_stream<T, VEC>(p + i);
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) unpack2<T, VEC>(v, e, x[i + 2 * e], x[i + 2 * e + 1]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = Elem<T>::to_f(p[e]);
  }
}

// The larger / smaller of the two, NaN if either is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct Quantised {
  uint32_t codes;  // element e in bits 4e .. 4e + 3
  __half2 params;  // step, low
};

constexpr float kRounder = 12582912.f;  // 1.5 * 2^23: x + kRounder holds rint(x) in its low bits

// The four lanes of a group call this together.
__device__ __forceinline__ Quantised quantise8(const float (&x)[8]) {
  float top = x[0], low = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    top = max_nan(top, x[e]);
    low = min_nan(low, x[e]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  Quantised r;
  r.params = __floats2half2_rn(__fmul_rn(__fsub_rn(top, low), 1.f / 15.f), low);
  // an infinity or a NaN among the elements leaves one here
  if (not_finite(*reinterpret_cast<const uint32_t*>(&r.params))) r.params = __float2half2_rn(__int_as_float(0x7fffffff));
  const float step = __low2float(r.params), base = __high2float(r.params);
  const float inv = step > 0.f ? __fdividef(1.f / 15.f, step) : 0.f;  // codes of 0 where there is no step
  float worst = 0.f, off[8];
  uint32_t word = 0, own = 0;  // own: the rounder's own bits, 0x4b400000 at every shift that keeps some
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    // the quotient over 15, clamped to 0 .. 1 on the way
    const float q = __saturatef(__fsub_rn(x[e], base) * inv), n = fmaf(q, 15.f, kRounder);
    off[e] = fabsf(fmaf(q, 15.f, -__fsub_rn(n, kRounder)));
    worst = fmaxf(worst, off[e]);
    word += __float_as_uint(n) << (4 * e);
    own += 0x4b400000u << (4 * e);
  }
  r.codes = word - own;
  constexpr float kTie = 0.5f - 1.f / 65536.f;
  if (worst > kTie) {
    // Exact ties are common in 16-bit data (one element in a thousand), so only those
    // close to one are done again.
    unsigned close = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) close |= off[e] > kTie ? 1u << e : 0u;
#pragma unroll 1
    while (close) {
      const int e = __ffs(close) - 1;
      close &= close - 1;
      float y = x[0];  // x[e], without an array in memory
#pragma unroll
      for (int i = 1; i < 8; ++i) y = i == e ? x[i] : y;
      const float n = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(y, base), step)), 0.f), 15.f);
      r.codes = (r.codes & ~(15u << (4 * e))) | (static_cast<uint32_t>(n) << (4 * e));
    }
  }
  return r;
}

// N 32-bit words next to each other.
template <int N>
__device__ __forceinline__ void put_words(void* p, const uint32_t (&w)[N]) {
  if constexpr (N == 4) *static_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (N == 2) *static_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else *static_cast<uint32_t*>(p) = w[0];
}
template <int N>
__device__ __forceinline__ void get_words(const void* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 x = *static_cast<const uint4*>(p);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else if constexpr (N == 2) {
    const uint2 x = *static_cast<const uint2*>(p);
    w[0] = x.x, w[1] = x.y;
  } else {
    w[0] = *static_cast<const uint32_t*>(p);
  }
}

template <typename T, bool PACKS, int N>
__global__ void __launch_bounds__(256) kv4_append_kernel(const __grid_constant__ Kv4RowsArgs a) {
  const int G = a.c.D / kKv4Group;
  const unsigned quad = blockIdx.x * 64u + (threadIdx.x >> 2);
  const int c = threadIdx.x & 3;
  const unsigned total = static_cast<unsigned>(a.B) * a.T * a.c.heads * (G / N);
  const bool live = quad < total;  // whole groups; the shuffles need every lane
  const GroupRef at = group_ref<N>(a, live ? quad : 0);
  const long long row = live ? kv4_row(a, at) : -1;
  float k[N][8] = {}, v[N][8] = {};
  if (row >= 0) {
    const int e = at.g * kKv4Group + c * 8;
    const T* kr = static_cast<const T*>(a.k) + at.b * a.ks[0] + at.t * a.ks[1] + at.h * a.ks[2] + e;
    const T* vr = static_cast<const T*>(a.v) + at.b * a.vs[0] + at.t * a.vs[1] + at.h * a.vs[2] + e;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      load8<T, PACKS>(kr + i * kKv4Group, k[i]);
      load8<T, PACKS>(vr + i * kKv4Group, v[i]);
    }
  }
  Quantised qk[N], qv[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    qk[i] = quantise8(k[i]);
    qv[i] = quantise8(v[i]);
  }
  if (row < 0) {
    if (row == -2) atomicOr(&g_kv4_status, kStatusCacheRange);
    return;
  }
  unsigned char* kc = static_cast<unsigned char*>(a.c.k_codes) + row * (a.c.D / 2);
  uint16_t* vc = reinterpret_cast<uint16_t*>(static_cast<unsigned char*>(a.c.v_codes) + row * (a.c.D / 2));
  uint32_t words[N], params[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    words[i] = qk[i].codes;
    const __half2 p = c == 0 ? qk[i].params : qv[i].params;
    params[i] = *reinterpret_cast<const uint32_t*>(&p);
  }
  put_words<N>(reinterpret_cast<uint32_t*>(kc) + c * G + at.g, words);
  if constexpr (N == 1) {
    vc[2 * c * G + at.g] = static_cast<uint16_t>(qv[0].codes);
    vc[(2 * c + 1) * G + at.g] = static_cast<uint16_t>(qv[0].codes >> 16);
  } else {
    uint32_t lower[N / 2], upper[N / 2];  // the groups' half words r = 2 c and 2 c + 1
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      lower[i] = __byte_perm(qv[2 * i].codes, qv[2 * i + 1].codes, 0x5410);
      upper[i] = __byte_perm(qv[2 * i].codes, qv[2 * i + 1].codes, 0x7632);
    }
    put_words<N / 2>(vc + 2 * c * G + at.g, lower);
    put_words<N / 2>(vc + (2 * c + 1) * G + at.g, upper);
  }
  if (c < 2) put_words<N>(static_cast<uint32_t*>(c == 0 ? a.c.k_params : a.c.v_params) + row * G + at.g, params);
}

// Codes become floats by way of 2^23 + n (an exact difference; conversion instructions are
// an eighth as fast).
template <typename T>
__device__ __forceinline__ void store_values(T* out, uint32_t codes, __half2 params, bool there) {
  const float step = there ? __low2float(params) : 0.f, low = there ? __high2float(params) : 0.f;
  constexpr int VEC = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8; i += VEC) {
    Pack<T, VEC> y;
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
      float v[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t n = ((codes >> (4 * (i + e + j))) & 15u) | 0x4b000000u;
        v[j] = fmaf(step, __uint_as_float(n) - 8388608.f, low);
      }
      if constexpr (std::is_same<T, float>::value) {
        y.e[e] = v[0];
        y.e[e + 1] = v[1];
      } else if constexpr (std::is_same<T, __half>::value) {
        *reinterpret_cast<__half2*>(&y.e[e]) = __floats2half2_rn(v[0], v[1]);
      } else {
        *reinterpret_cast<__nv_bfloat162*>(&y.e[e]) = __floats2bfloat162_rn(v[0], v[1]);
      }
    }
    __stcs(reinterpret_cast<uint4*>(out + i), *reinterpret_cast<const uint4*>(&y));
  }
}

template <typename T, int N>
__global__ void __launch_bounds__(256) kv4_read_kernel(const __grid_constant__ Kv4RowsArgs a) {
  const int G = a.c.D / kKv4Group;
  const unsigned quad = blockIdx.x * 64u + (threadIdx.x >> 2);
  const int c = threadIdx.x & 3;
  if (quad >= static_cast<unsigned>(a.B) * a.T * a.c.heads * (G / N)) return;
  const GroupRef at = group_ref<N>(a, quad);
  const long long row = kv4_row(a, at);
  uint32_t kw[N] = {}, vw[N] = {}, kp[N] = {}, vp[N] = {};
  if (row >= 0) {
    const unsigned char* kc = static_cast<const unsigned char*>(a.c.k_codes) + row * (a.c.D / 2);
    const uint16_t* vc = reinterpret_cast<const uint16_t*>(static_cast<const unsigned char*>(a.c.v_codes) + row * (a.c.D / 2));
    get_words<N>(reinterpret_cast<const uint32_t*>(kc) + c * G + at.g, kw);
    get_words<N>(static_cast<const uint32_t*>(a.c.k_params) + row * G + at.g, kp);
    get_words<N>(static_cast<const uint32_t*>(a.c.v_params) + row * G + at.g, vp);
    if constexpr (N == 1) {
      vw[0] = vc[2 * c * G + at.g] | (static_cast<uint32_t>(vc[(2 * c + 1) * G + at.g]) << 16);
    } else {
      uint32_t lower[N / 2], upper[N / 2];
      get_words<N / 2>(vc + 2 * c * G + at.g, lower);
      get_words<N / 2>(vc + (2 * c + 1) * G + at.g, upper);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        vw[2 * i] = __byte_perm(lower[i], upper[i], 0x5410);
        vw[2 * i + 1] = __byte_perm(lower[i], upper[i], 0x7632);
      }
    }
  } else if (row == -2) {
    atomicOr(&g_kv4_status, kStatusCacheRange);
  }
  const long long to = static_cast<long long>(quad) * (N * kKv4Group) + c * 8;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    store_values<T>(static_cast<T*>(a.k_out) + to + i * kKv4Group, kw[i], *reinterpret_cast<const __half2*>(&kp[i]), row >= 0);
    store_values<T>(static_cast<T*>(a.v_out) + to + i * kKv4Group, vw[i], *reinterpret_cast<const __half2*>(&vp[i]), row >= 0);
  }
}

namespace {

// Groups a thread, of those that a head has a multiple of: two to write (24006 tokens of 8
// heads of 128: 42 us; with four 48, the elements of four take registers that keep other
// warps away), four to read (18.9 us; with two 23.9).
int groups_a_thread(const Kv4RowsArgs& a, int most) {
  const int G = a.c.D / kKv4Group;
  return most == 4 && G % 4 == 0 ? 4 : (G % 2 == 0 ? 2 : 1);
}

unsigned blocks_of(const Kv4RowsArgs& a, int groups) {
  const long long threads = 4LL * a.B * a.T * a.c.heads * (a.c.D / kKv4Group / groups);
  return static_cast<unsigned>((threads + 255) / 256);
}

template <typename T>
cudaError_t append_t(const Kv4RowsArgs& a, cudaStream_t st) {
  bool packs = (reinterpret_cast<uintptr_t>(a.k) & 15u) == 0 && (reinterpret_cast<uintptr_t>(a.v) & 15u) == 0;
  for (int i = 0; i < 3; ++i) packs = packs && a.ks[i] * sizeof(T) % 16 == 0 && a.vs[i] * sizeof(T) % 16 == 0;
  const int n = groups_a_thread(a, 2);
  const auto fn = packs ? (n == 2 ? kv4_append_kernel<T, true, 2> : kv4_append_kernel<T, true, 1>)
                        : (n == 2 ? kv4_append_kernel<T, false, 2> : kv4_append_kernel<T, false, 1>);
  fn<<<blocks_of(a, n), 256, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t read_t(const Kv4RowsArgs& a, cudaStream_t st) {
  const int n = groups_a_thread(a, 4);
  const auto fn = n == 4 ? kv4_read_kernel<T, 4> : n == 2 ? kv4_read_kernel<T, 2> : kv4_read_kernel<T, 1>;
  fn<<<blocks_of(a, n), 256, 0, st>>>(a);
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
  switch (dtype) {
    case ATTNRES_DTYPE_F32: return read_t<float>(a, st);
    case ATTNRES_DTYPE_F16: return read_t<__half>(a, st);
    default: return read_t<__nv_bfloat16>(a, st);
  }
}

cudaError_t read_kv4_status(unsigned* status, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_kv4_status, sizeof(unsigned));
  if (e != cudaSuccess || !reset) return e;
  const unsigned zero = 0;
  return cudaMemcpyToSymbol(g_kv4_status, &zero, sizeof(unsigned));
}

}  // namespace attnres
