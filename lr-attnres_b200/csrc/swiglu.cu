// Gated projection of the model's MLP: with W = [Wv; Wg] ([2F, C], the value rows
// first) and x [N, C],
//   u = x Wv^T,  g = x Wg^T,  h = u * silu(g),  silu(g) = g * sigmoid(g)
// Backward, from x, W and dh:
//   du = dh silu(g),  dg = dh u sigmoid(g) (1 + g (1 - sigmoid(g)))
//   dx = du Wv + dg Wg,   dW = [du^T x; dg^T x]
//
// All three products are tiles of one tensor-core kernel (tcgen05, operands by TMA,
// fp32 accumulators in tensor memory):
//   gate forward   A = x rows, B = 128 value rows and the same 128 gate rows of W: a
//                  tile holds u and g of the same outputs, so the activation and the
//                  product are its epilogue and neither u nor g reaches memory;
//   gate backward  the same products again, and from them, with dh, du and dg,
//                  rounded once to the data's type for the two products that follow.
//                  (Keeping u and g from the forward instead costs 4NF bytes of memory a
//                  layer and two more roundings in the gradients; it saves one of the
//                  step's four products.)
//   dx             A = [du dg] rows, B = W (K index slow: MN-major operand);
//   dW             A = [du dg]^T, B = x, both MN-major.
// Few tokens: swiglu_few_kernel streams W once past the registers of all SMs.
//
// Roles in a CTA: warp 0 one thread of TMA loads into a ring of stages, warp 1 one
// thread of tcgen05.mma, 8 warps of epilogue on the other half of the accumulators.
// Every mbarrier wait is bounded (~2 s, a status bit on timeout); tensor memory is
// always released.
#include <algorithm>

#include "common.cuh"
#include "launch_cache.h"
#include "mma.cuh"
#include "swiglu.h"
#include "tma.cuh"
#include "umma.cuh"

namespace attnres {

static __device__ unsigned int g_swiglu_status = 0;

constexpr int kGmM = 128, kGmN = 256, kGmK = 64;  // tile, and columns of a stage
constexpr int kGmStages = 4;
constexpr uint32_t kGmABytes = kGmM * kGmK * 2, kGmBBytes = kGmN * kGmK * 2;
constexpr uint32_t kGmStageBytes = kGmABytes + kGmBBytes;
constexpr int kGmEpiWarps = 8;
constexpr int kGmThreads = (2 + kGmEpiWarps) * 32;
constexpr size_t kGmSmem = 1024 + kGmStages * kGmStageBytes + 256;

enum GemmMode { kGateForward, kGateBackward, kGradInput, kGradWeight };

struct GemmArgs {
  CUtensorMap a, b, b2;  // b2: the gate rows of the two gate modes
  void* out;             // h [N, F]; [du dg] [N, 2F]; dx [N, C]; dW [2F, C]
  const void* dh;        // gate backward
  long long out_stride, dh_stride;
  long long M;           // rows of the output
  int cols;              // columns of the output (gate modes: F)
  int tiles_m, tiles_n, ksteps;
  uint32_t idesc;
};

// Tiles in bands of 16 row tiles, rows fastest inside a band: the CTAs running at one
// time read few distinct row and column panels, which stay in L2.
__device__ __forceinline__ void tile_at(const GemmArgs& a, int tile, int& m, int& n) {
  constexpr int BAND = 16;
  const int per_band = BAND * a.tiles_n, band = tile / per_band, in = tile - band * per_band;
  const int rows = min(BAND, a.tiles_m - band * BAND);
  n = in / rows;
  m = band * BAND + in - n * rows;
}

__device__ __forceinline__ float sigmoid_fast(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v) {
  Pack<T, 8> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value)
      reinterpret_cast<__half2*>(r.e)[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    else
      reinterpret_cast<__nv_bfloat162*>(r.e)[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  }
  *reinterpret_cast<Pack<T, 8>*>(p) = r;
}

template <typename T, int MODE>
__global__ void __launch_bounds__(kGmThreads, 1) swiglu_gemm_kernel(const __grid_constant__ GemmArgs a) {
  constexpr bool GATE = MODE == kGateForward || MODE == kGateBackward;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* stages =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(stages + kGmStages * kGmStageBytes);
  uint64_t* empty = full + kGmStages;
  uint64_t* acc_full = empty + kGmStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* done = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ntiles = a.tiles_m * a.tiles_n, nk = a.ksteps;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kGmStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], kGmEpiWarps);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ---------------- TMA producer -------------------------------------------
    if (lane == 0) {
      long long it = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < ntiles && ok; tile += gridDim.x) {
        int m, n;
        tile_at(a, tile, m, n);
        for (int kc = 0; kc < nk; ++kc, ++it) {
          const int st = static_cast<int>(it % kGmStages);
          if (*abort_flag || !mbar_wait_bounded(&empty[st], static_cast<uint32_t>((it / kGmStages) & 1) ^ 1u)) {
            atomicOr(&g_swiglu_status, kStatusEmptyWaitTimeout);
            *abort_flag = 1;
            ok = false;
            break;
          }
          unsigned char* sa = stages + st * kGmStageBytes;
          unsigned char* sb = sa + kGmABytes;
          mbar_arrive_expect_tx(&full[st], kGmStageBytes);
          if (MODE == kGradWeight) {
            for (int i = 0; i < kGmM / 64; ++i)
              tma_load_2d(sa + i * 64 * 128, &a.a, m * kGmM + i * 64, kc * kGmK, &full[st]);
          } else {
            tma_load_2d(sa, &a.a, kc * kGmK, m * kGmM, &full[st]);
          }
          if (GATE) {
            tma_load_2d(sb, &a.b, kc * kGmK, n * 128, &full[st]);
            tma_load_2d(sb + 128 * 128, &a.b2, kc * kGmK, n * 128, &full[st]);
          } else {
            for (int i = 0; i < kGmN / 64; ++i)
              tma_load_2d(sb + i * 64 * 128, &a.b, n * kGmN + i * 64, kc * kGmK, &full[st]);
          }
        }
      }
      if (!ok) {
        for (long long j = (it > kGmStages ? it - kGmStages : 0); j < it; ++j)
          if (!mbar_wait_bounded(&full[j % kGmStages], static_cast<uint32_t>((j / kGmStages) & 1)))
            atomicOr(&g_swiglu_status, kStatusDrainTimeout);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer -----------------------------------------------
    if (lane == 0) {
      long long it = 0;
      int count = 0;
      bool issued_any = false;
      for (int tile = blockIdx.x; tile < ntiles; tile += gridDim.x, ++count) {
        const int ab = count & 1;
        if (*abort_flag || !mbar_wait_bounded(&acc_empty[ab], static_cast<uint32_t>((count >> 1) & 1) ^ 1u)) {
          atomicOr(&g_swiglu_status, kStatusEmptyWaitTimeout);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t acc = tmem + ab * kGmN;
        bool ok = true;
        for (int kc = 0; kc < nk; ++kc, ++it) {
          const int st = static_cast<int>(it % kGmStages);
          if (*abort_flag || !mbar_wait_bounded(&full[st], static_cast<uint32_t>((it / kGmStages) & 1))) {
            atomicOr(&g_swiglu_status, kStatusFullWaitTimeout);
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const unsigned char* sa = stages + st * kGmStageBytes;
          const unsigned char* sb = sa + kGmABytes;
          // K = 16 an instruction: 32 bytes on in a K-major tile, two groups of 8
          // rows (2048 bytes) in an MN-major one
          const uint64_t da = MODE == kGradWeight ? umma_desc_sw128_mn(sa, 64 * 128) : umma_desc_sw128(sa);
          const uint64_t db = GATE ? umma_desc_sw128(sb) : umma_desc_sw128_mn(sb, 64 * 128);
#pragma unroll
          for (int k = 0; k < kGmK / 16; ++k)
            umma_f16(acc, da + (MODE == kGradWeight ? 128 : 2) * k, db + (GATE ? 2 : 128) * k, a.idesc,
                     (kc > 0 || k > 0) ? 1u : 0u);
          umma_commit(&empty[st]);
          issued_any = true;
        }
        if (!ok) break;
        umma_commit(&acc_full[ab]);
      }
      umma_commit(done);  // all MMAs of this CTA retired before the accumulators are freed
      if (issued_any && !mbar_wait_bounded(done, 0)) atomicOr(&g_swiglu_status, kStatusDrainTimeout);
    }
  } else {
    // ---------------- epilogue: one accumulator row a thread, half the columns a warp
    const int q = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lane_off = static_cast<uint32_t>(q * 32) << 16;
    T* out = static_cast<T*>(a.out);
    int count = 0;
    for (int tile = blockIdx.x; tile < ntiles; tile += gridDim.x, ++count) {
      int m, n;
      tile_at(a, tile, m, n);
      const int ab = count & 1;
      if (*abort_flag || !mbar_wait_bounded(&acc_full[ab], static_cast<uint32_t>((count >> 1) & 1))) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const long long row = static_cast<long long>(m) * kGmM + q * 32 + lane;
      const uint32_t acc = tmem + lane_off + ab * kGmN;
      if constexpr (GATE) {
        const int f0 = n * 128 + half * 64;
        T* o = out + row * a.out_stride + f0;
        const T* dh = MODE == kGateBackward ? static_cast<const T*>(a.dh) + row * a.dh_stride + f0 : nullptr;
#pragma unroll 1
        for (int c = 0; c < 64; c += 16) {
          uint32_t ur[16], gr[16];
          tmem_ld16_nowait(acc + half * 64 + c, ur);
          tmem_ld16_nowait(acc + 128 + half * 64 + c, gr);
          Pack<T, 8> d[2];
          if (MODE == kGateBackward) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (row < a.M && f0 + c + i * 8 < a.cols) d[i] = load_stream<T, 8>(dh + c + i * 8);
              else d[i] = Pack<T, 8>{};
          }
          tmem_ld_wait();
          tmem_regs_ready(ur);
          tmem_regs_ready(gr);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float y[8], z[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float u = __uint_as_float(ur[i * 8 + e]), g = __uint_as_float(gr[i * 8 + e]);
              const float s = sigmoid_fast(g), silu = g * s;
              if (MODE == kGateForward) {
                y[e] = u * silu;
              } else {
                const float dhe = Elem<T>::to_f(d[i].e[e]);
                y[e] = dhe * silu;
                z[e] = dhe * u * (s + silu * (1.f - s));
              }
            }
            if (row < a.M && f0 + c + i * 8 < a.cols) {
              store8<T>(o + c + i * 8, y);
              if (MODE == kGateBackward) store8<T>(o + a.cols + c + i * 8, z);
            }
          }
        }
      } else {
        const int c0 = n * kGmN + half * 128;
        T* o = out + row * a.out_stride + c0;
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
          uint32_t r0[16], r1[16];
          tmem_ld16_nowait(acc + half * 128 + c, r0);
          tmem_ld16_nowait(acc + half * 128 + c + 16, r1);
          tmem_ld_wait();
          tmem_regs_ready(r0);
          tmem_regs_ready(r1);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (row < a.M && c0 + c + i * 8 < a.cols) {
              float y[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(i < 2 ? r0[i * 8 + e] : r1[(i - 2) * 8 + e]);
              store8<T>(o + c + i * 8, y);
            }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[ab]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// few tokens
// ---------------------------------------------------------------------------
// A CTA forms 8 outputs f of every token: the 8 value rows and 8 gate rows of W are
// the 16 rows of mma.sync.m16n8k16's A (u and g of one output then lie in the same
// thread), the tokens its 8 columns; its 8 warps split C, and their sums are added
// in order through shared memory. A lane takes 16 consecutive bytes of a row, the
// same from x: which of the 16 k a lane holds does not matter as long as A and B
// agree. Bound by reading W once; the tensor cores of this kernel idle most of the
// time, so the older instruction, whose operands come from registers, suffices.
constexpr int kFewWarps = 8;

struct FewArgs {
  const void *x, *w;
  void* h;
  long long x_stride, w_stride, h_stride;
  int N, C, F;
};

template <typename T, int NT>  // NT tiles of 8 tokens
__global__ void __launch_bounds__(kFewWarps * 32) swiglu_few_kernel(const __grid_constant__ FewArgs a) {
  __shared__ float sums[kFewWarps][NT][32][4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int f = blockIdx.x * 8 + r;  // F is a multiple of 8
  const T* wu = static_cast<const T*>(a.w) + f * a.w_stride + c * 8;
  const T* wg = wu + a.F * a.w_stride;
  const T* x = static_cast<const T*>(a.x) + r * a.x_stride + c * 8;
  float acc[NT][4] = {};
  constexpr int DEPTH = 4;  // loads of W in flight: 4 x 32 columns
  for (int k0 = warp * 32; k0 < a.C; k0 += kFewWarps * 32 * DEPTH) {
    uint4 u[DEPTH], g[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int k = k0 + d * kFewWarps * 32;
      u[d] = g[d] = make_uint4(0, 0, 0, 0);
      if (k + c * 8 < a.C) {
        const Pack<T, 8> pu = load_stream<T, 8>(wu + k), pg = load_stream<T, 8>(wg + k);
        u[d] = *reinterpret_cast<const uint4*>(&pu);
        g[d] = *reinterpret_cast<const uint4*>(&pg);
      }
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int k = k0 + d * kFewWarps * 32;
      if (k >= a.C) break;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        uint4 b = make_uint4(0, 0, 0, 0);
        if (r + 8 * t < a.N && k + c * 8 < a.C) b = *reinterpret_cast<const uint4*>(x + 8 * t * a.x_stride + k);
        mma_16816<T>(acc[t], u[d].x, g[d].x, u[d].y, g[d].y, b.x, b.y);
        mma_16816<T>(acc[t], u[d].z, g[d].z, u[d].w, g[d].w, b.z, b.w);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) *reinterpret_cast<float4*>(sums[warp][t][lane]) = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 64; i += kFewWarps * 32) {
    // output f of token n: u in register e of lane (f, n / 2), g in register 2 + e
    const int fo = i & 7, n = i >> 3, t = n >> 3, e = n & 1, from = fo * 4 + ((n & 7) >> 1);
    if (n >= a.N) break;
    float u = 0.f, g = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      u += sums[w][t][from][e];
      g += sums[w][t][from][2 + e];
    }
    static_cast<T*>(a.h)[n * a.h_stride + blockIdx.x * 8 + fo] = Elem<T>::from_f(u * (g * sigmoid_fast(g)));
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
namespace {

constexpr int kFewTokens = 32;

template <typename T>
cudaError_t few_t(const SwigluArgs& s, cudaStream_t st) {
  FewArgs a{s.x, s.w, s.out, s.x_stride, s.w_stride, s.F, static_cast<int>(s.N), s.C, s.F};
  const unsigned grid = s.F / 8;
  if (s.N <= 8) swiglu_few_kernel<T, 1><<<grid, kFewWarps * 32, 0, st>>>(a);
  else if (s.N <= 16) swiglu_few_kernel<T, 2><<<grid, kFewWarps * 32, 0, st>>>(a);
  else swiglu_few_kernel<T, 4><<<grid, kFewWarps * 32, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename T, int MODE>
cudaError_t gemm_t(GemmArgs& a, int dtype, cudaStream_t st) {
  constexpr bool GATE = MODE == kGateForward || MODE == kGateBackward;
  a.tiles_m = static_cast<int>((a.M + kGmM - 1) / kGmM);
  a.tiles_n = GATE ? ceil_div_i(a.cols, 128) : ceil_div_i(a.cols, kGmN);
  a.idesc = umma_idesc_f16(dtype == ATTNRES_DTYPE_BF16, MODE == kGradWeight, !GATE, kGmM, kGmN);
  const void* fn = reinterpret_cast<const void*>(&swiglu_gemm_kernel<T, MODE>);
  cudaError_t e = ensure_dynamic_smem(fn, static_cast<int>(kGmSmem));
  int nsm = 0;
  if (e == cudaSuccess) e = cached_sm_count(&nsm);
  if (e != cudaSuccess) return e;
  const int grid = std::min(a.tiles_m * a.tiles_n, nsm);
  swiglu_gemm_kernel<T, MODE><<<grid, kGmThreads, kGmSmem, st>>>(a);
  return cudaGetLastError();
}

constexpr cudaError_t kNoTensorMap = cudaErrorInvalidValue;

// Tensor map of a [rows, cols] matrix read in boxes of 64 columns x box_rows. The
// driver call needs a context in the calling thread, which a thread of the autograd
// engine that has made no runtime call yet lacks: cudaSetDevice binds it.
bool map(CUtensorMap* m, int dtype, const void* p, long long rows, int cols, long long stride, int box_rows) {
  if (encode_2d(m, dtype, p, rows, cols, stride, box_rows)) return true;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return false;
  return encode_2d(m, dtype, p, rows, cols, stride, box_rows);
}

template <typename T>
cudaError_t gate_t(const SwigluArgs& s, bool backward, int dtype, cudaStream_t st) {
  GemmArgs a{};
  const T* w = static_cast<const T*>(s.w);
  if (!map(&a.a, dtype, s.x, s.N, s.C, s.x_stride, kGmM) || !map(&a.b, dtype, w, s.F, s.C, s.w_stride, 128) ||
      !map(&a.b2, dtype, w + s.F * s.w_stride, s.F, s.C, s.w_stride, 128))
    return kNoTensorMap;
  a.M = s.N;
  a.cols = s.F;
  a.ksteps = ceil_div_i(s.C, kGmK);
  if (!backward) {
    a.out = s.out;
    a.out_stride = s.F;
    return gemm_t<T, kGateForward>(a, dtype, st);
  }
  a.out = s.workspace;
  a.out_stride = 2LL * s.F;
  a.dh = s.dh;
  a.dh_stride = s.dh_stride;
  return gemm_t<T, kGateBackward>(a, dtype, st);
}

template <typename T>
cudaError_t backward_t(const SwigluArgs& s, int dtype, cudaStream_t st) {
  cudaError_t e = gate_t<T>(s, true, dtype, st);
  if (e != cudaSuccess) return e;
  const int F2 = 2 * s.F;
  if (s.dx) {
    GemmArgs a{};
    if (!map(&a.a, dtype, s.workspace, s.N, F2, F2, kGmM) || !map(&a.b, dtype, s.w, F2, s.C, s.w_stride, kGmK))
      return kNoTensorMap;
    a.out = s.dx;
    a.out_stride = s.C;
    a.M = s.N;
    a.cols = s.C;
    a.ksteps = ceil_div_i(F2, kGmK);
    if ((e = gemm_t<T, kGradInput>(a, dtype, st)) != cudaSuccess) return e;
  }
  if (s.dw) {
    GemmArgs a{};
    if (!map(&a.a, dtype, s.workspace, s.N, F2, F2, kGmK) || !map(&a.b, dtype, s.x, s.N, s.C, s.x_stride, kGmK))
      return kNoTensorMap;
    a.out = s.dw;
    a.out_stride = s.C;
    a.M = F2;
    a.cols = s.C;
    a.ksteps = static_cast<int>((s.N + kGmK - 1) / kGmK);
    if ((e = gemm_t<T, kGradWeight>(a, dtype, st)) != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t swiglu_launch(bool backward, int dtype, const SwigluArgs& s, cudaStream_t st) {
  const bool bf16 = dtype == ATTNRES_DTYPE_BF16;
  if (backward) return bf16 ? backward_t<__nv_bfloat16>(s, dtype, st) : backward_t<__half>(s, dtype, st);
  if (s.N <= kFewTokens) return bf16 ? few_t<__nv_bfloat16>(s, st) : few_t<__half>(s, st);
  return bf16 ? gate_t<__nv_bfloat16>(s, false, dtype, st) : gate_t<__half>(s, false, dtype, st);
}

cudaError_t read_swiglu_status(unsigned* status, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_swiglu_status, sizeof(unsigned));
  if (e != cudaSuccess || !reset) return e;
  const unsigned zero = 0;
  return cudaMemcpyToSymbol(g_swiglu_status, &zero, sizeof(unsigned));
}

}  // namespace attnres
