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
// Two CTAs of a cluster share a tile (tcgen05 cta_group::2): each loads its own 128 rows
// of A and half of B and holds its 128 rows of the sums, so an SM takes in 32 KB for 128 x
// 256 x 64 products instead of 48. With one CTA a tile the products ran at 1185 TFLOP/s,
// bound by that intake.
// Roles: warp 0 one thread of TMA loads into a ring of stages, warp 1 of the even CTA one
// thread of tcgen05.mma for both, 8 warps of epilogue on the other half of the
// accumulators. Every mbarrier wait is bounded (~2 s, a status bit on timeout); tensor
// memory is always released.
// 16384 tokens, 1024 -> 4096, bf16: gate forward 188 us (1465 TFLOP/s), gate backward 222
// (1240; its epilogue moves 400 MB), dx and dW 365 (1505). The tensor cores are busy 84 to
// 89 % of the cycles (gate backward 65 %) and the power limit holds the clock at 1.6 GHz.
#include <algorithm>

#include "cluster.cuh"
#include "common.cuh"
#include "launch_cache.h"
#include "mma.cuh"
#include "swiglu.h"
#include "tma.cuh"
#include "umma.cuh"

namespace attnres {

static __device__ unsigned int g_swiglu_status = 0;

constexpr int kGmM = 256, kGmK = 64;  // rows of a pair's tile, columns of a stage
constexpr int kGmBuf = 32 * 128;      // 32 rows x 64 outputs of an epilogue warp
constexpr int kGmEpiWarps = 8;
constexpr int kGmThreads = (2 + kGmEpiWarps) * 32;
constexpr int kGmShared = 7 * 32768;  // bytes of the ring and of the epilogue's buffers
constexpr size_t kGmSmem = 1024 + kGmShared + 512;

enum GemmMode { kGateForward, kGateBackward, kGradients };

// One product: out [M, cols] = A B, in tiles of 256 x BN.
struct GemmJob {
  CUtensorMap a, b, b2;  // b2: the gate rows of the two gate modes
  CUtensorMap out, out2;  // h [N, F], or du and dg as [N, F] inside [N, 2F]; dW [2F, C]; dx [N, C]
  bool wanted;
  long long M;
  int cols;              // columns of the output (gate modes: F)
  int tiles_m, tiles_n, ksteps;
  uint32_t idesc;
};
struct GemmArgs {
  GemmJob job[2];  // kGradients: dW, then dx; else one
  CUtensorMap dh;  // gate backward: [N, F]
  // kGradients: the tiles of job `first` (the one with the longer sums) are dealt out in
  // turn; then come the other job's, x each for the first `more` pairs (which have one of
  // the long ones more than the others), y each for the rest
  int first, more, x, y;
};

struct TileRef {
  int job, m, n;
};

// Tiles in bands of 8 row tiles, rows fastest inside a band: the pairs running at one
// time read few distinct row and column panels, which stay in L2.
__device__ __forceinline__ TileRef tile_at(const GemmArgs& a, int job, int tile) {
  constexpr int BAND = 8;
  const GemmJob& g = a.job[job];
  const int per_band = BAND * g.tiles_n, band = tile / per_band, in = tile - band * per_band;
  const int rows = min(BAND, g.tiles_m - band * BAND), n = in / rows;
  return {job, band * BAND + in - n * rows, n};
}

// The i-th tile of pair p of P, job -1 when there is none.
template <int MODE>
__device__ __forceinline__ TileRef tile_of(const GemmArgs& a, int p, int P, int i) {
  const int first = MODE == kGradients ? a.first : 0;
  const int count = a.job[first].tiles_m * a.job[first].tiles_n;
  const int own = p < count ? (count - 1 - p) / P + 1 : 0;
  if (i < own) return tile_at(a, first, p + i * P);
  if (MODE == kGradients) {
    const GemmJob& other = a.job[1 - first];
    const int j = i - own, each = p < a.more ? a.x : a.y;
    const int tile = p < a.more ? j * a.more + p : a.more * a.x + j * (P - a.more) + p - a.more;
    if (j < each && tile < other.tiles_m * other.tiles_n) return tile_at(a, 1 - first, tile);
  }
  return {-1, 0, 0};
}

// ---- the two-CTA forms of the tensor-core instructions
// A TMA load into this CTA's shared memory that completes on an mbarrier of the cluster's
// even CTA (its shared::cluster address).
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void umma_f16_pair(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      :
      : "r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
// Arrives on the mbarrier at this address in both CTAs when the MMAs issued so far are done.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
// Arrives on an mbarrier of a CTA of the cluster (shared::cluster address).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ float sigmoid_fast(float g) { return __fdividef(1.f, 1.f + __expf(-g)); }

// Where 16-byte piece `piece` of row `row` lies in a 128-byte-swizzled buffer.
__device__ __forceinline__ unsigned char* piece_at(unsigned char* buf, int row, int piece) {
  return buf + row * 128 + ((piece ^ (row & 7)) << 4);
}

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

// The ring's waits. The producer and the issuer are one thread each and every cycle of
// their loops counts (a stage of a narrow tile is 256 cycles of products), so the usual
// case is one test and nothing else; only a wait that has to go on looks at the abort
// flag and the clock.
__device__ __forceinline__ bool ring_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool ring_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (ring_test(bar, parity)) return true;
  const unsigned long long t0 = global_timer_ns();
  while (!ring_test(bar, parity))
    if (*abort_flag || global_timer_ns() - t0 > kWaitLimitNs) return ring_test(bar, parity);
  return true;
}

template <typename T, int MODE, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGmThreads, 1)
    swiglu_gemm_kernel(const __grid_constant__ GemmArgs a) {
  constexpr bool GATE = MODE != kGradients;
  // Bytes of each CTA: 64 columns of A and of B, and SUB of those a stage: a stage costs its
  // issuer 0.16 us besides the products, as much as those of 64 columns of a narrow tile
  // (wide tiles, dx and dW of 16384 tokens: 365 us with 128 columns a stage, 385 with 64).
  // (The gate backward's second output buffers leave its wide tiles no room for that.)
  constexpr int BUFS = MODE == kGateBackward ? 2 : 1, kRing = kGmShared - kGmEpiWarps * BUFS * kGmBuf;
  constexpr int SUB = BN == 128 || BUFS == 1 ? 2 : 1;
  constexpr uint32_t kA = 128 * kGmK * 2, kB = BN / 2 * kGmK * 2, kSub = kA + kB, kStage = SUB * kSub;
  constexpr int STAGES = kRing / kStage, F = BN / 2;                               // F: outputs of a gate tile
  // 64 columns a chunk; a gate tile of one chunk goes to either half of the epilogue warps in turn
  constexpr int CHUNKS = GATE ? F / 64 : BN / 64;
  constexpr bool ALTERNATE = CHUNKS == 1;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* stages =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* bufs = stages + kRing;  // [epilogue warps][BUFS] output buffers
  uint64_t* full = reinterpret_cast<uint64_t*>(bufs + kGmEpiWarps * BUFS * kGmBuf);  // the even CTA's are used
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;  // the even CTA's are used
  uint64_t* done = acc_empty + 2;
  uint64_t* dh_full = done + 1;  // [epilogue warps]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(dh_full + kGmEpiWarps);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * (ALTERNATE ? kGmEpiWarps / 2 : kGmEpiWarps));
    }
    mbar_init(done, 1);
    for (int i = 0; i < kGmEpiWarps; ++i) mbar_init(&dh_full[i], 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ---------------- TMA producer: this CTA's half of each stage ------------------
    if (lane == 0) {
      const uint32_t full0 = map_to_rank(smem_u32(full), 0), empty0 = smem_u32(empty);
      int st = 0;
      long long posted = 0;
      uint32_t phase = 1;  // an untouched barrier's previous phase counts as done
      bool ok = true;
      for (int i = 0; ok; ++i) {
        const TileRef t = tile_of<MODE>(a, pair, pairs, i);
        if (t.job < 0) break;
        const GemmJob& g = a.job[t.job];
        const int m0 = t.m * kGmM + rank * 128, n0 = GATE ? t.n * F : t.n * BN + rank * (BN / 2);
        const CUtensorMap* const bmap = GATE && rank ? &g.b2 : &g.b;
        const int k_end = g.ksteps * kGmK;
        for (int k0 = 0; k0 < k_end; k0 += SUB * kGmK) {
          if (!ring_wait(empty0 + 8 * st, phase, abort_flag)) {
            atomicOr(&g_swiglu_status, kStatusEmptyWaitTimeout);
            *abort_flag = 1;
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full[st], 2 * kStage);
          const uint32_t bar = full0 + 8 * st;
#pragma unroll
          for (int sub = 0; sub < SUB; ++sub) {  // past the end of K: zeros
            unsigned char* sa = stages + st * kStage + sub * kSub;
            unsigned char* sb = sa + kA;
            const int k = k0 + sub * kGmK;
            if (GATE) {
              tma_load_2d_pair(sa, &g.a, k, m0, bar);
              tma_load_2d_pair(sb, bmap, k, n0, bar);
            } else {
              if (t.job == 0) {  // dW: rows of A are columns of [du dg]
                tma_load_2d_pair(sa, &g.a, m0, k, bar);
                tma_load_2d_pair(sa + 64 * 128, &g.a, m0 + 64, k, bar);
              } else {
                tma_load_2d_pair(sa, &g.a, k, m0, bar);
              }
#pragma unroll
              for (int j = 0; j < BN / 128; ++j) tma_load_2d_pair(sb + j * 64 * 128, bmap, n0 + j * 64, k, bar);
            }
          }
          ++posted;
          if (++st == STAGES) {
            st = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok && rank == 0) {
        // stages that were posted land in both CTAs before either goes on to exit
        for (long long j = (posted > STAGES ? posted - STAGES : 0); j < posted; ++j)
          if (!mbar_wait_bounded(&full[j % STAGES], static_cast<uint32_t>((j / STAGES) & 1)))
            atomicOr(&g_swiglu_status, kStatusDrainTimeout);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer of the pair ---------------------------------------
    if (lane == 0 && rank == 0) {
      const uint32_t full0 = smem_u32(full);
      // K = 16 an instruction: 32 bytes on in a K-major tile, two groups of 8 rows (2048
      // bytes) in an MN-major one
      const uint64_t k_major = umma_desc_sw128(stages), mn_major = umma_desc_sw128_mn(stages, 64 * 128);
      constexpr uint64_t kStageStep = kStage >> 4;
      const uint64_t b0 = (GATE ? k_major : mn_major) + (kA >> 4);
      constexpr uint64_t b_step = GATE ? 2 : 128;
      int st = 0;
      uint32_t phase = 0;
      bool issued_any = false, ok = true;
      for (int i = 0; ok; ++i) {
        const TileRef t = tile_of<MODE>(a, pair, pairs, i);
        if (t.job < 0) break;
        const GemmJob& g = a.job[t.job];
        const int ab = i & 1;
        if (*abort_flag || !mbar_wait_cluster(&acc_empty[ab], static_cast<uint32_t>((i >> 1) & 1) ^ 1u)) {
          atomicOr(&g_swiglu_status, kStatusEmptyWaitTimeout);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t acc = tmem + ab * BN, idesc = g.idesc;
        const bool a_mn = !GATE && t.job == 0;
        const uint64_t a0 = a_mn ? mn_major : k_major, a_step = a_mn ? 128 : 2;
        const int steps = (g.ksteps + SUB - 1) / SUB;
        for (int k = 0; k < steps; ++k) {
          if (!ring_wait(full0 + 8 * st, phase, abort_flag)) {
            atomicOr(&g_swiglu_status, kStatusFullWaitTimeout);
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int sub = 0; sub < SUB; ++sub) {
            const uint64_t da = a0 + st * kStageStep + sub * (kSub >> 4), db = b0 + st * kStageStep + sub * (kSub >> 4);
#pragma unroll
            for (int j = 0; j < kGmK / 16; ++j)
              umma_f16_pair(acc, da + a_step * j, db + b_step * j, idesc, (k > 0 || sub > 0 || j > 0) ? 1u : 0u);
          }
          umma_commit_pair(&empty[st]);
          issued_any = true;
          if (++st == STAGES) {
            st = 0;
            phase ^= 1u;
          }
        }
        if (ok) umma_commit_pair(&acc_full[ab]);
      }
      umma_commit_pair(done);  // all MMAs retired before the accumulators are freed
      if (issued_any && !mbar_wait_bounded(done, 0)) atomicOr(&g_swiglu_status, kStatusDrainTimeout);
    }
  } else {
    // ---------------- epilogue: one accumulator row a thread, 64 columns at a time ----
    // into the warp's swizzled buffers, which TMA stores from (rows and columns past the
    // end are dropped there); dh comes the same way, a tile ahead.
    const int q = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lane_off = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t freed[2] = {map_to_rank(smem_u32(&acc_empty[0]), 0), map_to_rank(smem_u32(&acc_empty[1]), 0)};
    unsigned char* buf0 = bufs + (warp - 2) * BUFS * kGmBuf;
    unsigned char* buf1 = buf0 + (BUFS - 1) * kGmBuf;
    uint64_t* dh_bar = &dh_full[warp - 2];
    const int row0 = rank * 128 + q * 32, step = ALTERNATE ? 2 : 1;
    auto fetch_dh = [&](const TileRef& t) {  // lane 0, once buf0 is free
      mbar_arrive_expect_tx(dh_bar, kGmBuf);
      tma_load_2d(buf0, &a.dh, t.n * F + (ALTERNATE ? 0 : half * 64), t.m * kGmM + row0, dh_bar);
    };
    TileRef t = tile_of<MODE>(a, pair, pairs, ALTERNATE ? half : 0);
    if (MODE == kGateBackward && t.job >= 0 && lane == 0) fetch_dh(t);
    uint32_t dh_phase = 0;
    bool dh_pending = MODE == kGateBackward && t.job >= 0;
    for (int i = ALTERNATE ? half : 0; t.job >= 0; i += step) {
      const GemmJob& g = a.job[t.job];
      const int ab = i & 1;
      bool ok = !*abort_flag && mbar_wait_bounded(&acc_full[ab], static_cast<uint32_t>((i >> 1) & 1));
      if (MODE == kGateBackward && ok) {
        ok = mbar_wait_bounded(dh_bar, dh_phase);
        if (ok) {
          dh_pending = false;
          dh_phase ^= 1u;
        }
      }
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0) atomicOr(&g_swiglu_status, kStatusFullWaitTimeout);
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const uint32_t acc = tmem + lane_off + ab * BN;
      const int r0 = t.m * kGmM + row0;
      const TileRef next = tile_of<MODE>(a, pair, pairs, i + step);
      if constexpr (GATE) {
        const int chunk = ALTERNATE ? 0 : half;
#pragma unroll 1
        for (int c = 0; c < 64; c += 16) {
          uint32_t ur[16], gr[16];
          tmem_ld16_nowait(acc + chunk * 64 + c, ur);
          tmem_ld16_nowait(acc + F + chunk * 64 + c, gr);
          tmem_ld_wait();
          tmem_regs_ready(ur);
          tmem_regs_ready(gr);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            unsigned char* at = piece_at(buf0, lane, c / 8 + j);
            Pack<T, 8> d = {};
            if (MODE == kGateBackward) d = *reinterpret_cast<const Pack<T, 8>*>(at);
            float y[8], z[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float u = __uint_as_float(ur[j * 8 + e]), gt = __uint_as_float(gr[j * 8 + e]);
              const float s = sigmoid_fast(gt), silu = gt * s;
              if (MODE == kGateForward) {
                y[e] = u * silu;
              } else {
                const float dhe = Elem<T>::to_f(d.e[e]);
                y[e] = dhe * silu;
                z[e] = dhe * u * (s + silu * (1.f - s));
              }
            }
            store8<T>(reinterpret_cast<T*>(at), y);
            if (MODE == kGateBackward) store8<T>(reinterpret_cast<T*>(piece_at(buf1, lane, c / 8 + j)), z);
          }
        }
        tc_fence_before();
        fence_async_shared();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_cluster(freed[ab]);
          const int c0 = t.n * F + chunk * 64;
          if (c0 < g.cols && r0 < g.M) {
            tma_store_2d(&g.out, c0, r0, buf0);
            if (MODE == kGateBackward) tma_store_2d(&g.out2, c0, r0, buf1);
          }
          bulk_commit_group();
          bulk_wait_group_read0();
          if (MODE == kGateBackward && next.job >= 0) fetch_dh(next);
        }
        if (MODE == kGateBackward) dh_pending = next.job >= 0;
        __syncwarp();
      } else {
#pragma unroll 1
        for (int k = 0; k < CHUNKS / 2; ++k) {
          const int chunk = half * (CHUNKS / 2) + k;
#pragma unroll
          for (int c = 0; c < 64; c += 32) {
            uint32_t r[2][16];
            tmem_ld16_nowait(acc + chunk * 64 + c, r[0]);
            tmem_ld16_nowait(acc + chunk * 64 + c + 16, r[1]);
            tmem_ld_wait();
            tmem_regs_ready(r[0]);
            tmem_regs_ready(r[1]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float y[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(r[j >> 1][(j & 1) * 8 + e]);
              store8<T>(reinterpret_cast<T*>(piece_at(buf0, lane, c / 8 + j)), y);
            }
          }
          if (k == CHUNKS / 2 - 1) tc_fence_before();
          fence_async_shared();
          __syncwarp();
          if (lane == 0) {
            if (k == CHUNKS / 2 - 1) mbar_arrive_cluster(freed[ab]);
            const int c0 = t.n * BN + chunk * 64;
            if (c0 < g.cols && r0 < g.M) tma_store_2d(&g.out, c0, r0, buf0);
            bulk_commit_group();
            bulk_wait_group_read0();
          }
          __syncwarp();
        }
      }
      t = next;
    }
    if (lane == 0) {
      // a load of dh still in flight lands before the CTA's shared memory is given away
      if (dh_pending && !mbar_wait_bounded(dh_bar, dh_phase)) atomicOr(&g_swiglu_status, kStatusDrainTimeout);
      bulk_wait_group0();
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves while the other's MMAs or arrivals may reach it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
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
// 1024 -> 4096 in bf16, 16.8 MB: 5.1 us at 1 token, 6.6 at 12, 8.2 at 27.
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
  // Steps of 32 columns whose loads are in flight together. x's loads go with W's from two
  // token tiles on (in the product's loop instead they cost 1024 -> 4096 at 12 tokens 8.2 us
  // instead of 6.6, at 27 9.0 instead of 8.6; at 1 token 5.1 instead of 5.5).
  constexpr int DEPTH = NT == 4 ? 2 : 4;
  constexpr bool AHEAD = NT > 1;
  for (int k0 = warp * 32; k0 < a.C; k0 += kFewWarps * 32 * DEPTH) {
    uint4 u[DEPTH], g[DEPTH], b[DEPTH][NT];
    auto load_x = [&](int k, uint4 (&to)[NT]) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        to[t] = make_uint4(0, 0, 0, 0);
        if (r + 8 * t < a.N && k + c * 8 < a.C) to[t] = *reinterpret_cast<const uint4*>(x + 8 * t * a.x_stride + k);
      }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int k = k0 + d * kFewWarps * 32;
      u[d] = g[d] = make_uint4(0, 0, 0, 0);
      if (k + c * 8 < a.C) {
        const Pack<T, 8> pu = load_stream<T, 8>(wu + k), pg = load_stream<T, 8>(wg + k);
        u[d] = *reinterpret_cast<const uint4*>(&pu);
        g[d] = *reinterpret_cast<const uint4*>(&pg);
      }
      if (AHEAD) load_x(k, b[d]);
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int k = k0 + d * kFewWarps * 32;
      if (k >= a.C) break;
      if (!AHEAD) load_x(k, b[d]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        mma_16816<T>(acc[t], u[d].x, g[d].x, u[d].y, g[d].y, b[d][t].x, b[d][t].y);
        mma_16816<T>(acc[t], u[d].z, g[d].z, u[d].w, g[d].w, b[d][t].z, b[d][t].w);
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

// Up to here the streaming kernel: 1024 -> 4096 at 32 tokens 8.4 us against 12.0 on tiles,
// at 12 tokens 6.7 against 12.0.
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

// Time of a list of tiles on P pairs, in steps of 64 columns of a 256 x 256 tile (0.42 us).
// A step of a 256 x 128 tile counts 0.75: 0.5 alone, but it has 3/4 of the loads and twice
// the starts and ends for its products (1531 tokens, 776 -> 2056, gate forward: 19.1 us on
// wide tiles, 20.0 on narrow ones; dx, 42 narrow tiles or 24 wide: 21.7 and 28 us).
double tiles_cost(const GemmJob& g, int BN, bool gate, int P) {
  const int n = gate ? ceil_div_i(g.cols, BN / 2) : ceil_div_i(g.cols, BN);
  const long long tiles = static_cast<long long>((g.M + kGmM - 1) / kGmM) * n;
  return static_cast<double>((tiles + P - 1) / P) * g.ksteps * (BN == 256 ? 1.0 : 0.75);
}

template <typename T, int MODE, int BN>
cudaError_t gemm_bn(GemmArgs& a, int dtype, int pairs, cudaStream_t st) {
  constexpr bool GATE = MODE != kGradients;
  long long tiles = 0;
  int count[2] = {0, 0};
  for (int i = 0; i < 2; ++i) {
    GemmJob& g = a.job[i];
    if (!g.wanted) continue;  // no tiles
    g.tiles_m = static_cast<int>((g.M + kGmM - 1) / kGmM);
    g.tiles_n = GATE ? ceil_div_i(g.cols, BN / 2) : ceil_div_i(g.cols, BN);
    g.idesc = umma_idesc_f16(dtype == ATTNRES_DTYPE_BF16, !GATE && i == 0, !GATE, kGmM, BN);
    count[i] = g.tiles_m * g.tiles_n;
    tiles += count[i];
  }
  const int P = static_cast<int>(std::min<long long>(tiles, pairs));
  if (MODE == kGradients) {
    // the split of the shorter tiles that ends soonest: near the even share of all the work
    a.first = a.job[0].wanted && (!a.job[1].wanted || a.job[0].ksteps >= a.job[1].ksteps) ? 0 : 1;
    const int n0 = count[a.first], n1 = count[1 - a.first];
    a.more = n0 % P;
    if (n1 > 0) {
      const double k0 = a.job[a.first].ksteps, k1 = a.job[1 - a.first].ksteps, base = n0 / P * k0;
      const double even = (n0 * k0 + n1 * k1) / P;
      const int guess = std::max(0, static_cast<int>((even - base - k0) / k1));
      double best = -1.0;
      for (int x = std::max(0, guess - 2); x <= guess + 2; ++x) {
        const long long left = std::max<long long>(0, n1 - static_cast<long long>(a.more) * x);
        const int y = static_cast<int>((left + P - a.more - 1) / (P - a.more));
        const double end = std::max(a.more > 0 ? base + k0 + x * k1 : 0.0, base + y * k1);
        if (best < 0.0 || end < best) {
          best = end;
          a.x = x;
          a.y = y;
        }
      }
    }
  }
  const void* fn = reinterpret_cast<const void*>(&swiglu_gemm_kernel<T, MODE, BN>);
  const cudaError_t e = ensure_dynamic_smem(fn, static_cast<int>(kGmSmem));
  if (e != cudaSuccess) return e;
  swiglu_gemm_kernel<T, MODE, BN><<<2 * P, kGmThreads, kGmSmem, st>>>(a);
  return cudaGetLastError();
}

// Operand tiles of both widths read boxes of 64 rows or columns of B, so the maps do not
// depend on the width; the gate modes' boxes are BN / 2 rows.
template <typename T, int MODE>
cudaError_t gemm_t(GemmArgs& a, int dtype, int pairs, bool wide, cudaStream_t st) {
  return wide ? gemm_bn<T, MODE, 256>(a, dtype, pairs, st) : gemm_bn<T, MODE, 128>(a, dtype, pairs, st);
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

// Pairs of CTAs that are resident at once (one CTA an SM; a group of SMs with an odd one
// leaves it out): a persistent launch of more would queue the rest behind all the work.
cudaError_t pair_count(int* pairs) {
  const void* fn = reinterpret_cast<const void*>(&swiglu_gemm_kernel<__nv_bfloat16, kGateForward, 256>);
  cudaError_t e = ensure_dynamic_smem(fn, static_cast<int>(kGmSmem));
  if (e == cudaSuccess) e = cached_max_clusters(pairs, fn, 2, kGmThreads, kGmSmem);
  if (e == cudaSuccess && *pairs < 1) e = cudaErrorInvalidConfiguration;
  return e;
}

template <typename T>
cudaError_t gate_t(const SwigluArgs& s, bool backward, int dtype, cudaStream_t st) {
  int pairs = 0;
  const cudaError_t e = pair_count(&pairs);
  if (e != cudaSuccess) return e;
  GemmArgs a{};
  GemmJob& g = a.job[0];
  g.M = s.N;
  g.cols = s.F;
  g.ksteps = ceil_div_i(s.C, kGmK);
  const bool wide = tiles_cost(g, 256, true, pairs) <= tiles_cost(g, 128, true, pairs);
  const T* w = static_cast<const T*>(s.w);
  if (!map(&g.a, dtype, s.x, s.N, s.C, s.x_stride, 128) || !map(&g.b, dtype, w, s.F, s.C, s.w_stride, wide ? 128 : 64) ||
      !map(&g.b2, dtype, w + s.F * s.w_stride, s.F, s.C, s.w_stride, wide ? 128 : 64))
    return kNoTensorMap;
  g.wanted = true;
  if (!backward) {
    if (!map(&g.out, dtype, s.out, s.N, s.F, s.F, 32)) return kNoTensorMap;
    return gemm_t<T, kGateForward>(a, dtype, pairs, wide, st);
  }
  T* d = static_cast<T*>(s.workspace);
  if (!map(&g.out, dtype, d, s.N, s.F, 2LL * s.F, 32) || !map(&g.out2, dtype, d + s.F, s.N, s.F, 2LL * s.F, 32) ||
      !map(&a.dh, dtype, s.dh, s.N, s.F, s.dh_stride, 32))
    return kNoTensorMap;
  return gemm_t<T, kGateBackward>(a, dtype, pairs, wide, st);
}

template <typename T>
cudaError_t backward_t(const SwigluArgs& s, int dtype, cudaStream_t st) {
  cudaError_t e = gate_t<T>(s, true, dtype, st);
  if (e != cudaSuccess) return e;
  int pairs = 0;
  if ((e = pair_count(&pairs)) != cudaSuccess) return e;
  const int F2 = 2 * s.F;
  GemmArgs a{};
  double cost[2] = {0.0, 0.0};  // of wide and narrow tiles
  if (s.dw) {
    GemmJob& g = a.job[0];
    if (!map(&g.a, dtype, s.workspace, s.N, F2, F2, kGmK) || !map(&g.b, dtype, s.x, s.N, s.C, s.x_stride, kGmK) ||
        !map(&g.out, dtype, s.dw, F2, s.C, s.C, 32))
      return kNoTensorMap;
    g.wanted = true;
    g.M = F2;
    g.cols = s.C;
    g.ksteps = static_cast<int>((s.N + kGmK - 1) / kGmK);
    cost[0] += tiles_cost(g, 256, false, pairs);
    cost[1] += tiles_cost(g, 128, false, pairs);
  }
  if (s.dx) {
    GemmJob& g = a.job[1];
    if (!map(&g.a, dtype, s.workspace, s.N, F2, F2, 128) || !map(&g.b, dtype, s.w, F2, s.C, s.w_stride, kGmK) ||
        !map(&g.out, dtype, s.dx, s.N, s.C, s.C, 32))
      return kNoTensorMap;
    g.wanted = true;
    g.M = s.N;
    g.cols = s.C;
    g.ksteps = ceil_div_i(F2, kGmK);
    cost[0] += tiles_cost(g, 256, false, pairs);
    cost[1] += tiles_cost(g, 128, false, pairs);
  }
  return gemm_t<T, kGradients>(a, dtype, pairs, cost[0] <= cost[1], st);
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
