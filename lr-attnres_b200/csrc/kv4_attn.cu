// Attention of new query tokens over the 4-bit paged cache (format: kv4.h).
//
//   z_j = scale <q, k_j>, k_j = low_j + step_j n_j (a group of 32 elements at a time)
//   out = sum_j softmax(z)_j v_j over the places j that the token may see
// Token t of a sequence with `length` keys and `count` new tokens stands at place
// length - count + t and sees the places up to its own. Query head h reads key head
// h / (Hq / Hkv): the query heads of one key head, times the new tokens, are the rows
// that share one pass over its keys. A row that sees nothing gives zeros: its sum of
// weights is 0 (as that of a row whose finite scores all overflow fp32 to -inf). A row with
// a score that is NaN, or with an infinity or NaN in its query, is NaN by its sum; the
// maximum alone does not tell (comparisons drop NaN, so it stays -inf over NaN scores).
//
// One pass with the running maximum and sum of the softmax. The products run on
// mma.sync with the cache as the 16-row operand and the query rows as its 8 columns
// (one token of one head fills one column: the tensor cores have time to spare, HBM has
// not). Both multiply f16. A logic operation takes two codes out of a word:
//   scores  the bits n and n << 4 alone are f16's small numbers 2^-24 n and 2^-20 n; q is
//           scaled by a power of two per row (its largest element to 2^10 .. 2^11), and by
//           16 more where it meets the smaller ones, so its elements are exact down to
//           2^-24 of the largest. z = step * sum_d q_d n_d + low Q, Q the sum of the
//           group's q: exact products, fp32 sums
//   output  0x6400 | n is 1024 + n and 0x5400 | n << 4 is 64 + n; the difference to 1024 or
//           64 is exact, step n + low is rounded once to f16, and so are the weights (for f16
//           outputs they are the sum of two f16 numbers: one rounding less of the output's
//           own size). Weights below f16's normal range, 2^-14, are off by up to 2^-25 either
//           way; a warp's weights are relative to its own maximum over at most 1024 places,
//           so this adds up to less than 2^-15 of the largest
// The row of a key is an accumulator's row and a value's column: weights change sides
// by movmatrix. Keys are taken in the order i ^ ((i >> 1) & 1) so that lanes that differ
// in their keys read different halves of the banks.
//
// A value that some rows may not see must not reach them as 0 * NaN: in the stage
// around a sequence's end, values that nobody sees count as zero, and so do groups with
// an infinity or NaN, which are written into the sums of the rows that do see them as the
// NaN that any weight for them makes, 0 included. Groups whose largest value lies beyond
// f16 (finite step and low reach 2^20) are multiplied in units of 2^5. A stage takes the
// longer way that looks at all this if it lies around an end or its value params ask for it.
//
// A CTA takes a stretch of places of one (sequence, key head, 8 NT query rows); its four
// warps walk through it 32 or 64 places at a time, each with a ring of its own that bulk
// copies fill (codes and params of 16 places are contiguous in a page). Sums of
// the warps are joined in shared memory, those of the stretches by kv4_join_kernel.
// Every mbarrier wait is bounded (~2 s, a status bit on timeout).
//
// HBM is the floor (40 bytes a place of 64 elements, keys and values each): 8 sequences of
// 50000 places, 16 heads of 64, 3 tokens: 158 us with the join for 512 MB (3.2 TB/s); 8 x
// 50000 places, 8 heads of 128, 4 query heads each: 134 us (3.8 TB/s). No unit is full there
// (logic pipe 61 %, issue slots 61 %, DRAM 34 %, tensor cores 15 %): with the 16 or 20 warps
// an SM that the registers leave, a quarter of its places, the steps of a stage wait for one
// another. A stretch of a few stages is mostly its start and end: 24 ragged sequences up to
// 6000 places of 8 heads of 128 32 us for 72 MB. The look at each stage's value params costs
// 1 to 3 % of these times.
#include <algorithm>

#include "common.cuh"
#include "kv4.h"
#include "launch_cache.h"
#include "mma.cuh"
#include "tma.cuh"

namespace attnres {

static __device__ unsigned int g_kv4_attn_status = 0;

constexpr int kAtWarps = 4;
// Places of a stage, and stages of a warp's ring: what a stage costs besides its places
// (the wait, the copies, the maximum's vote) is a third of 32 places' work at head_dim 64.
constexpr int at_keys(int D) { return D == 64 ? 64 : 32; }
constexpr int at_stages(int) { return 2; }
constexpr bool at_shared_q(int D) { return D == 128; }
constexpr int kAtMaxStretch = 4096;
constexpr float kLog2e = 1.4426950408889634f;
// The running maximum is raised only when a score passes it by this much (in powers of
// two): weights then reach 2^kSlack, far from f16's 2^16, and almost every step goes
// without the shuffles and the rescaling.
constexpr float kSlack = 8.f;

struct AttnLaunch {
  Kv4AttnArgs a;
  int group, rows, row_tiles;  // query heads a key head; rows = T * group; tiles of 8 NT rows
  int q_packs;                 // q's rows start on 16-byte boundaries
  int stretch, splits;         // places of a CTA, stretches of the longest possible sequence
  float* part_o;               // [B, heads, row_tiles, splits, 8 NT, D]
  float2* part_ml;             // [B, heads, row_tiles, splits, 8 NT]
};

// Code pair k of a word (bits 4 k and 16 + 4 k) in the f16 halves' bits 0 .. 3 (even k) or
// 4 .. 7 (odd k); and with the exponent that makes them 1024 + n or 64 + n.
__device__ __forceinline__ uint32_t code_bits(uint32_t w, int k) {
  return (k >= 2 ? w >> 8 : w) & ((k & 1) ? 0x00f000f0u : 0x000f000fu);
}
__device__ __forceinline__ uint32_t code_off(int k) { return (k & 1) ? 0x54005400u : 0x64006400u; }
constexpr float kOddUnit = 1.f / 1048576.f;  // 2^-20: a code in bits 4 .. 7

__device__ __forceinline__ uint32_t half_sub(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t half_fma(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                            *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t half_mul(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t half_pack(float a, float b) {
  const __half2 r = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&r);
}
// The largest values of two groups, low + 15 step: rounded to f16 they are infinite or NaN if
// one leaves it. steps, lows: the groups' params, taken apart.
__device__ __forceinline__ __half2 largest_values(uint32_t steps, uint32_t lows) {
  const uint32_t top = half_fma(steps, 0x4b804b80u, lows);
  return __habs2(*reinterpret_cast<const __half2*>(&top));
}
// Whether one of four groups has a value beyond f16 or none at all.
__device__ __forceinline__ bool leave_f16(__half2 a, __half2 b) {
  const uint32_t inf = 0x7c007c00u;
  return !__hblt2(__hmax2_nan(a, b), *reinterpret_cast<const __half2*>(&inf));
}
// The same over the value params of a stage, four groups a lane.
__device__ __forceinline__ bool stage_leaves_f16(const unsigned char* params, int lane) {
  const uint4 p = *reinterpret_cast<const uint4*>(params + lane * 16);
  return __any_sync(0xffffffffu, leave_f16(largest_values(__byte_perm(p.x, p.y, 0x5410u), __byte_perm(p.x, p.y, 0x7632u)),
                                           largest_values(__byte_perm(p.z, p.w, 0x5410u), __byte_perm(p.z, p.w, 0x7632u))));
}

__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// (a0, a1) += (b0, b1) and (a0, a1) *= (b0, b1) in packed fp32.
__device__ __forceinline__ void add_pair(float& a0, float& a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "add.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(b0), "f"(b1));
}
__device__ __forceinline__ void mul_pair(float& a0, float& a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
      "mul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
      : "+f"(a0), "+f"(a1)
      : "f"(b0), "f"(b1));
}

// G words at p, as one load where the size allows.
template <int G>
__device__ __forceinline__ void load_words(const unsigned char* p, uint32_t (&w)[G]) {
  if constexpr (G == 4) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
  } else if constexpr (G == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x, w[1] = x.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

enum StageKind { kPlain, kMasked, kCareful };
template <StageKind K>
using Kind = std::integral_constant<StageKind, K>;

// Sequence b's keys and new tokens, and how many of the keys its page table can hold.
struct SeqFacts {
  int length, count, held;
};
__device__ __forceinline__ SeqFacts seq_facts(const Kv4AttnArgs& a, int b) {
  SeqFacts s;
  s.length = max(a.lengths[b], 0);
  s.held = min(s.length, a.max_pages * a.c.page);  // the host refuses tables of more than 2^30 places
  s.count = a.counts ? min(max(a.counts[b], 0), a.T) : a.T;
  return s;
}
// The places that a token sees: 0 .. last (negative: none).
__device__ __forceinline__ int last_place(const SeqFacts& s, int t) {
  return t < s.count ? s.length - s.count + t : -1;
}

// Where a row's outputs lie, in rows of head_dim.
__device__ __forceinline__ long long out_index(const AttnLaunch& L, int b, int h, int row) {
  const int t = row / L.group, head = h * L.group + row - t * L.group;
  return (static_cast<long long>(b) * L.a.T + t) * L.a.Hq + head;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kAtWarps * 32, NT == 1 ? (D == 64 ? 5 : 4) : 2) kv4_attn_kernel(const __grid_constant__ AttnLaunch L) {
  constexpr int G = D / kKv4Group, HALF = D / 2;
  constexpr int KEYS = at_keys(D), PIECES = KEYS / 16, STAGES = at_stages(D);
  constexpr int kCode = KEYS * HALF, kParam = KEYS * G * 4;  // bytes of a stage
  constexpr int kStage = 2 * (kCode + kParam);
  constexpr int ROWS = 8 * NT;
  const Kv4AttnArgs& a = L.a;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(16) int rows16[kAtMaxStretch / 16];  // row of the pool / 16 of each 16 places, -1 where there is no page
  __shared__ uint64_t bars[kAtWarps][STAGES];
  __shared__ float warp_m[kAtWarps][ROWS], warp_l[kAtWarps][ROWS], row_top[ROWS], row_sum[ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x % L.splits, tile = blockIdx.x / L.splits, h = blockIdx.y, b = blockIdx.z;
  // this thread's first entry of the page table, on its way while the length is read
  const int from = split * L.stretch, first_slot = (from + static_cast<int>(threadIdx.x) * 16) / a.c.page;
  const int first_page = first_slot < a.max_pages ? a.table[b * a.table_stride + first_slot] : -1;
  const SeqFacts seq = seq_facts(a, b);
  const int to = min(from + L.stretch, seq.held);
  if (from == 0 && threadIdx.x == 0 && seq.held < seq.length) atomicOr(&g_kv4_attn_status, kStatusCacheRange);
  // the join may take up its place on the GPU; it waits for this grid's end before it reads
  if (L.splits > 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (from >= to && L.splits > 1) return;  // the join knows how many stretches there are

  const int count = (to - from + KEYS - 1) / KEYS;  // a warp's stages: its number, + 4, ...
  for (int i = threadIdx.x; i < count * PIECES; i += kAtWarps * 32) {
    if (i * 16 >= to - from) {
      rows16[i] = -1;
      continue;
    }
    const int at = from + i * 16, slot = at / a.c.page;
    const int p = i < kAtWarps * 32 ? first_page : a.table[b * a.table_stride + slot];
    const bool there = p >= 0 && p < a.c.pages;
    if (!there) atomicOr(&g_kv4_attn_status, kStatusCacheRange);
    const int place16 = (at - slot * a.c.page) >> 4;
    rows16[i] = there ? static_cast<int>((static_cast<long long>(p) * a.c.heads + h) * (a.c.page >> 4)) + place16 : -1;
  }
  if (lane == 0)
    for (int i = 0; i < STAGES; ++i) mbar_init(&bars[warp][i], 1);
  fence_mbar_init();
  __syncthreads();

  unsigned char* ring = smem + warp * STAGES * kStage;
  // Lanes copy 16 places each: lane & 3 is keys, key params, values, value params.
  const unsigned char* const my_src = static_cast<const unsigned char*>(
      (lane & 2) ? ((lane & 1) ? a.c.v_params : a.c.v_codes) : ((lane & 1) ? a.c.k_params : a.c.k_codes));
  const uint32_t my_bytes = 16 * ((lane & 1) ? G * 4 : HALF);
  const int my_piece = lane >> 2;
  unsigned char* const my_dst = ring + ((lane & 1) ? 2 * kCode + ((lane >> 1) & 1) * kParam : ((lane >> 1) & 1) * kCode) +
                                my_piece * my_bytes;
  auto fetch = [&](int stage, int slot) {
    const int r = my_piece < PIECES ? rows16[stage * PIECES + my_piece] : -1;
    const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, r >= 0)) * (kStage / PIECES / 4);
    if (lane == 0) {
      if (bytes) mbar_arrive_expect_tx(&bars[warp][slot], bytes);
      else mbar_arrive(&bars[warp][slot]);
    }
    __syncwarp();
    if (r >= 0)
      bulk_g2s(my_dst + slot * kStage, my_src + static_cast<long long>(r) * my_bytes, my_bytes, &bars[warp][slot]);
  };
#pragma unroll
  for (int i = 0; i < STAGES; ++i)
    if (warp + i * kAtWarps < count) fetch(warp + i * kAtWarps, i);

  // the query rows as the second operand: column g of tile j is row 8 j + g. At head_dim
  // 128 they lie in shared memory, where the four warps share them: with them in registers
  // three CTAs fit on an SM, and the kernel waits for its own latencies.
  constexpr bool SHARED_Q = at_shared_q(D);
  __shared__ uint4 q_shared[SHARED_Q ? NT * G * 32 : 1];
  uint32_t qf[SHARED_Q ? 1 : NT][SHARED_Q ? 1 : G][4];
  float qsum[NT][G][2], zscale[NT][2];  // of rows 8 j + 2 c, 2 c + 1
  int last[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int row = tile * ROWS + 8 * j + g;
    const T* q = static_cast<const T*>(a.q);
    const bool there = row < L.rows;
    if (there) {
      const int t = row / L.group, head = h * L.group + row - t * L.group;
      q += b * a.qs[0] + t * a.qs[1] + head * a.qs[2];
    }
    float x[G][8], most = 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      Pack<T, 8> v = {};
      if (there && L.q_packs) {
        v = load_pack<T, 8>(q + i * 32 + c * 8);
      } else if (there) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v.e[k] = q[i * 32 + c * 8 + k];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[i][k] = Elem<T>::to_f(v.e[k]);
        most = fmaxf(most, fabsf(x[i][k]));
      }
    }
#pragma unroll
    for (int s = 1; s < 4; s <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, s));
    // 2^(10 - exponent of the largest element), from the exponent's bits. An infinity makes
    // the row NaN: its scores are infinite or NaN, and over infinite ones the softmax is NaN.
    const int exponent = __float_as_int(most) >> 23;
    const float up = exponent == 255 ? __int_as_float(0x7fffffff) : __int_as_float(min(264 - exponent, 250) << 23);
#pragma unroll
    for (int i = 0; i < G; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = (k & 1) ? up : 16.f * up;
        w[k] = half_pack(x[i][k] * f, x[i][k + 4] * f);
      }
      if constexpr (SHARED_Q) {
        if (warp == i % kAtWarps) q_shared[(j * G + i) * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) qf[j][i][k] = w[k];
      }
      float s[4] = {};
      const uint32_t one = 0x3c003c00u, sixteenth = 0x2c002c00u;
      mma_16816<__half>(s, sixteenth, sixteenth, one, one, w[0], w[1]);
      mma_16816<__half>(s, sixteenth, sixteenth, one, one, w[2], w[3]);
#pragma unroll
      for (int e = 0; e < 2; ++e) qsum[j][i][e] = s[e] * kOddUnit;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = tile * ROWS + 8 * j + 2 * c + e;
      last[j][e] = r < L.rows ? last_place(seq, r / L.group) : -1;
      zscale[j][e] = a.scale * (kLog2e / kOddUnit) / __shfl_sync(0xffffffffu, up, 4 * (2 * c + e));
    }
  }
  if constexpr (SHARED_Q) __syncthreads();
  int least = to - 1;  // places up to this one are seen by all rows that see any
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (tile * ROWS + 8 * j + 2 * c + e < L.rows) least = min(least, last[j][e]);
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, o));

  float o[NT][2 * G][4] = {}, m[NT][2], l[NT][2] = {};
#pragma unroll
  for (int j = 0; j < NT; ++j) m[j][0] = m[j][1] = -INFINITY;
  const int swap = (g >> 1) & 1;          // keys in the order i ^ ((i >> 1) & 1)
  // One stage, in three copies: as tests that are predicated away, what the rarer ones do
  // besides would take a third of the common one's issue slots. MASKED: some of its places
  // may not be seen by some row. CAREFUL: some value params, of any place, are not finite or
  // stand for values beyond f16 (in places that were not fetched, anything may).
  auto attend = [&](const unsigned char* kc, int at, int stage, auto kind) {
    constexpr bool MASKED = decltype(kind)::value != kPlain, CAREFUL = decltype(kind)::value == kCareful;
    const unsigned char* vc = kc + kCode;
    const unsigned char* kp = kc + 2 * kCode;
    const unsigned char* vp = kp + kParam;
    // ---- scores: accumulator row g (and g + 8) is a key, columns 2c, 2c + 1 rows
    float z[PIECES][NT][4];
#pragma unroll
    for (int mt = 0; mt < PIECES; ++mt) {
      const int key0 = mt * 16 + (g ^ swap), key1 = key0 + 8;
      uint32_t w0[G], w1[G], p0[G], p1[G];
      load_words<G>(kc + key0 * HALF + c * 4 * G, w0);
      load_words<G>(kc + key1 * HALF + c * 4 * G, w1);
      load_words<G>(kp + key0 * 4 * G, p0);
      load_words<G>(kp + key1 * 4 * G, p1);
#pragma unroll
      for (int i = 0; i < G; ++i) {
        uint32_t f0[4], f1[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f0[k] = code_bits(w0[i], k);
          f1[k] = code_bits(w1[i], k);
        }
        const float2 s0 = __half22float2(*reinterpret_cast<const __half2*>(&p0[i]));
        const float2 s1 = __half22float2(*reinterpret_cast<const __half2*>(&p1[i]));
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          uint4 w;
          if constexpr (SHARED_Q) w = q_shared[(j * G + i) * 32 + lane];
          else w = make_uint4(qf[j][i][0], qf[j][i][1], qf[j][i][2], qf[j][i][3]);
          float acc[4];
          mma_16816<__half>(acc, f0[0], f1[0], f0[1], f1[1], w.x, w.y, 0.f, 0.f, 0.f, 0.f);
          mma_16816<__half>(acc, f0[2], f1[2], f0[3], f1[3], w.z, w.w);
#pragma unroll
          for (int e = 0; e < 4; e += 2) {  // two rows at a time, in packed fp32
            const float2 s = e == 0 ? s0 : s1;
            float& z0 = z[mt][j][e];
            float& z1 = z[mt][j][e + 1];
            if (i == 0) mul2(z0, z1, s.y, qsum[j][i][0], qsum[j][i][1]);
            else fma2(z0, z1, s.y, qsum[j][i][0], qsum[j][i][1]);
            fma2(z0, z1, s.x, acc[e], acc[e + 1]);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (e % 2 == 0) mul_pair(z[mt][j][e], z[mt][j][e + 1], zscale[j][0], zscale[j][1]);
          if constexpr (MASKED) {
            const int place = at + (e < 2 ? key0 : key1);
            if (rows16[stage * PIECES + mt] < 0 || place >= to || place > last[j][e & 1]) z[mt][j][e] = -INFINITY;
          }
        }
    }

    // ---- running maximum; the sums o and l follow it
    bool passed = false;
    float top[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[j][e] = fmaxf(z[0][j][e], z[0][j][2 + e]);
#pragma unroll
        for (int mt = 1; mt < PIECES; ++mt) top[j][e] = fmaxf(top[j][e], fmaxf(z[mt][j][e], z[mt][j][2 + e]));
        passed |= top[j][e] > m[j][e] + kSlack;  // also the first score of a row: m is -inf
      }
    if (__any_sync(0xffffffffu, passed)) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float shrink[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int s = 4; s < 32; s <<= 1) top[j][e] = fmaxf(top[j][e], __shfl_xor_sync(0xffffffffu, top[j][e], s));
          const float mine = fmaxf(m[j][e], top[j][e]);
          shrink[e] = m[j][e] == mine ? 1.f : exp2_fast(m[j][e] - mine);
          m[j][e] = mine;
          l[j][e] *= shrink[e];
        }
#pragma unroll
        for (int i = 0; i < 2 * G; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[j][i][e] *= shrink[e & 1];
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const float less[2] = {m[j][0] == -INFINITY ? 0.f : -m[j][0], m[j][1] == -INFINITY ? 0.f : -m[j][1]};
#pragma unroll
      for (int mt = 0; mt < PIECES; ++mt)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          add_pair(z[mt][j][e], z[mt][j][e + 1], less[0], less[1]);
          z[mt][j][e] = exp2_fast(z[mt][j][e]);
          z[mt][j][e + 1] = exp2_fast(z[mt][j][e + 1]);
          add_pair(l[j][0], l[j][1], z[mt][j][e], z[mt][j][e + 1]);
        }
    }

    // ---- output: accumulator rows are elements of the value, columns query rows
#pragma unroll
    for (int mt = 0; mt < PIECES; ++mt) {
      uint32_t words[4][(G + 1) / 2], par[4][G];
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // MMA columns 2c, 2c + 1, 2c + 8, 2c + 9
        const int i = 2 * c + (k & 1), key = mt * 16 + (i ^ ((i >> 1) & 1)) + (k >> 1) * 8;
        load_words<(G + 1) / 2>(vc + key * HALF + g * 2 * G, words[k]);
        load_words<G>(vp + key * 4 * G, par[k]);
        if constexpr (MASKED) {
          const bool there = rows16[stage * PIECES + mt] >= 0 && at + key < to;
#pragma unroll
          for (int i2 = 0; i2 < G; ++i2)
            if (!there || (CAREFUL && not_finite(par[k][i2]))) par[k][i2] = 0;
        }
      }
      if constexpr (CAREFUL) {
        const int key0 = mt * 16 + (g ^ swap);
        uint32_t odd = 0;  // bit 4 e + i: group i of key key0 + 8 e has an infinity or NaN
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t mine[G];
          load_words<G>(vp + (key0 + 8 * e) * 4 * G, mine);
#pragma unroll
          for (int i = 0; i < G; ++i) odd |= static_cast<uint32_t>(not_finite(mine[i])) << (4 * e + i);
        }
        if (__any_sync(0xffffffffu, odd != 0)) {
          const int end = rows16[stage * PIECES + mt] >= 0 ? to : 0;
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              uint32_t seen = 0;  // groups of this lane's two keys that row 8 j + 2 c + r sees
              if (at + key0 < min(end, last[j][r] + 1)) seen |= odd & 15u;
              if (at + key0 + 8 < min(end, last[j][r] + 1)) seen |= odd >> 4;
#pragma unroll
              for (int i = 0; i < G; ++i)
                if (__ballot_sync(0xffffffffu, (seen >> i) & 1u) & (0x11111111u << c)) {
                  const float nan = __int_as_float(0x7fffffff);
                  o[j][2 * i][r] = o[j][2 * i][2 + r] = o[j][2 * i + 1][r] = o[j][2 * i + 1][2 + r] = nan;
                }
            }
        }
      }
      // the weights in f16; for f16 outputs also what that rounding left, as a second product:
      // the value's and the output's own roundings are of the same size there
      constexpr int PARTS = std::is_same<T, __half>::value ? 2 : 1;
      uint32_t pa[PARTS][NT], pb[PARTS][NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint32_t a0 = half_pack(z[mt][j][0], z[mt][j][1]), b0 = half_pack(z[mt][j][2], z[mt][j][3]);
        pa[0][j] = transposed(a0);
        pb[0][j] = transposed(b0);
        if constexpr (PARTS == 2) {
          const float2 a1 = __half22float2(*reinterpret_cast<const __half2*>(&a0));
          const float2 b1 = __half22float2(*reinterpret_cast<const __half2*>(&b0));
          pa[1][j] = transposed(half_pack(z[mt][j][0] - a1.x, z[mt][j][1] - a1.y));
          pb[1][j] = transposed(half_pack(z[mt][j][2] - b1.x, z[mt][j][3] - b1.y));
        }
      }
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const uint32_t pick = (i & 1) ? 0x7632u : 0x5410u;
        uint32_t f[2][4];
        uint32_t wa[PARTS][NT], wb[PARTS][NT];
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            wa[part][j] = pa[part][j];
            wb[part][j] = pb[part][j];
          }
        if constexpr (CAREFUL) {
          __half2 top[2];
#pragma unroll
          for (int e = 0; e < 2; ++e)
            top[e] = largest_values(__byte_perm(par[2 * e][i], par[2 * e + 1][i], 0x5410u),
                                    __byte_perm(par[2 * e][i], par[2 * e + 1][i], 0x7632u));
          if (__any_sync(0xffffffffu, leave_f16(top[0], top[1]))) {  // the values by 2^-5, the weights (up to 2^kSlack) by 2^5
#pragma unroll
            for (int k = 0; k < 4; ++k) par[k][i] = half_mul(par[k][i], 0x28002800u);
#pragma unroll
            for (int part = 0; part < PARTS; ++part)
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                wa[part][j] = half_mul(wa[part][j], 0x50005000u);
                wb[part][j] = half_mul(wb[part][j], 0x50005000u);
              }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // the pairs of keys 2c, 2c + 1 and 2c + 8, 2c + 9
          const uint32_t w = __byte_perm(words[2 * e][i >> 1], words[2 * e + 1][i >> 1], pick);
          const uint32_t step = __byte_perm(par[2 * e][i], par[2 * e + 1][i], 0x5410u);
          const uint32_t low = __byte_perm(par[2 * e][i], par[2 * e + 1][i], 0x7632u);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            f[e][k] = half_fma(half_sub(code_bits(w, k) | code_off(k), code_off(k)), step, low);
        }
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            mma_16816<__half>(o[j][2 * i], f[0][0], f[0][1], f[1][0], f[1][1], wa[part][j], wb[part][j]);
            mma_16816<__half>(o[j][2 * i + 1], f[0][2], f[0][3], f[1][2], f[1][3], wa[part][j], wb[part][j]);
          }
      }
    }
  };

  bool ok = true;
  int slot = 0, n = 0;
  uint32_t phase = 0;
  for (int stage = warp; stage < count; stage += kAtWarps, ++n) {
    ok = mbar_wait_bounded(&bars[warp][slot], phase);
    if (!__all_sync(0xffffffffu, ok)) {
      ok = false;
      break;
    }
    const int at = from + stage * KEYS;
    int rows = 0;  // negative if 16 places have no page
    if constexpr (PIECES == 4) {
      const int4 r = *reinterpret_cast<const int4*>(rows16 + stage * 4);
      rows = r.x | r.y | r.z | r.w;
    } else {
      const int2 r = *reinterpret_cast<const int2*>(rows16 + stage * 2);
      rows = r.x | r.y;
    }
    const unsigned char* const kc = ring + slot * kStage;
    if (stage_leaves_f16(kc + 2 * kCode + kParam, lane)) attend(kc, at, stage, Kind<kCareful>{});
    // nothing masked: places that are there and that every row sees
    else if (rows >= 0 && at + KEYS - 1 <= least) attend(kc, at, stage, Kind<kPlain>{});
    else attend(kc, at, stage, Kind<kMasked>{});
    __syncwarp();  // every lane has read the stage
    if (stage + STAGES * kAtWarps < count) fetch(stage + STAGES * kAtWarps, slot);
    if (++slot == STAGES) {
      slot = 0;
      phase ^= 1u;
    }
  }
  if (!ok) {
    if (lane == 0) atomicOr(&g_kv4_attn_status, kStatusFullWaitTimeout);
    // copies still in flight land before the CTA's shared memory is given away
    for (int i = 0; i < STAGES; ++i, ++n)
      if (warp + n * kAtWarps < count &&
          !mbar_wait_bounded(&bars[warp][n % STAGES], static_cast<uint32_t>((n / STAGES) & 1)) && lane == 0)
        atomicOr(&g_kv4_attn_status, kStatusDrainTimeout);
  }

  // ---- join the warps: l over the lanes of a column first
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int s = 4; s < 32; s <<= 1) {
#pragma unroll
      for (int e = 0; e < 2; ++e) l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], s);
    }
    if (g == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        warp_m[warp][8 * j + 2 * c + e] = m[j][e];
        warp_l[warp][8 * j + 2 * c + e] = l[j][e];
      }
    }
  }
  __syncthreads();  // every warp is done with its ring
  float* sums = reinterpret_cast<float*>(smem);  // [warps][ROWS][D + 4]
  constexpr int PITCH = D + 4;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 2 * G; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // element 32 (i / 2) + 4 g + 2 (i & 1) + (e / 2) of row 8 j + 2 c + (e & 1)
        const int element = 32 * (i >> 1) + 4 * g + 2 * (i & 1) + (e >> 1);
        sums[(warp * ROWS + 8 * j + 2 * c + (e & 1)) * PITCH + element] = o[j][i][e];
      }
  // weights of the warps' sums, once a row (over the maxima they came from)
  if (threadIdx.x < ROWS) {
    const int r = threadIdx.x;
    float top = warp_m[0][r], total = 0.f;
#pragma unroll
    for (int w = 1; w < kAtWarps; ++w) top = fmaxf(top, warp_m[w][r]);
#pragma unroll
    for (int w = 0; w < kAtWarps; ++w) {
      const float f = warp_m[w][r] == -INFINITY ? 0.f : exp2f(warp_m[w][r] - top);
      total += f * warp_l[w][r];
      warp_m[w][r] = f;
    }
    row_top[r] = top;
    row_sum[r] = total;
  }
  __syncthreads();
  const long long unit = ((static_cast<long long>(b) * a.c.heads + h) * L.row_tiles + tile) * L.splits + split;
  for (int i = threadIdx.x * 4; i < ROWS * D; i += kAtWarps * 32 * 4) {
    const int r = i / D, d = i - r * D, row = tile * ROWS + r;
    if (row >= L.rows) break;
    float y[4] = {};
#pragma unroll
    for (int w = 0; w < kAtWarps; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(&sums[(w * ROWS + r) * PITCH + d]);
      const float f = warp_m[w][r];
      y[0] += f * x.x, y[1] += f * x.y, y[2] += f * x.z, y[3] += f * x.w;
    }
    const float top = row_top[r], total = row_sum[r];
    if (L.splits == 1) {
      const long long to_row = out_index(L, b, h, row);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = total == 0.f ? 0.f : y[e] / total;
      store_pack<T, 4>(static_cast<T*>(a.out) + to_row * D + d, y);
      if (a.lse && d == 0) a.lse[to_row] = total == 0.f ? -INFINITY : (top + log2f(total)) / kLog2e;
    } else {
      store_pack<float, 4>(L.part_o + (unit * ROWS + r) * D + d, y);
      if (d == 0) L.part_ml[unit * ROWS + r] = make_float2(top, total);
    }
  }
}

// One CTA a row adds the stretches of its sequence: its warps take every fourth, and are
// added in order. (With a warp a row, one sequence of 100000 keys spent 60 of 103 us here,
// waiting for 196 loads one after the other.)
template <typename T, int D>
__global__ void __launch_bounds__(128) kv4_join_kernel(const __grid_constant__ AttnLaunch L, int tile_rows) {
  constexpr int VEC = D / 32;
  __shared__ float warp_top[4], warp_total[4], warp_sum_of[4][D];
  const Kv4AttnArgs& a = L.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = static_cast<int>(blockIdx.x % L.rows), bh = static_cast<int>(blockIdx.x / L.rows);
  const int h = bh % a.c.heads, b = bh / a.c.heads;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const SeqFacts seq = seq_facts(a, b);
  const int n = (seq.held + L.stretch - 1) / L.stretch;
  const long long first = (static_cast<long long>(bh) * L.row_tiles + row / tile_rows) * L.splits * tile_rows + row % tile_rows;
  const float2* ml = L.part_ml + first;  // of stretch s: s * tile_rows on
  const float* part = L.part_o + first * D + lane * VEC;
  float top = -INFINITY;
  for (int s = threadIdx.x; s < n; s += 128) top = fmaxf(top, ml[static_cast<long long>(s) * tile_rows].x);
  top = warp_max(top);
  if (lane == 0) warp_top[warp] = top;
  __syncthreads();
  top = fmaxf(fmaxf(warp_top[0], warp_top[1]), fmaxf(warp_top[2], warp_top[3]));
  float y[VEC] = {}, total = 0.f;
#pragma unroll 4
  for (int s = warp; s < n; s += 4) {
    const float2 x = ml[static_cast<long long>(s) * tile_rows];
    const Pack<float, VEC> p = load_pack<float, VEC>(part + static_cast<long long>(s) * tile_rows * D);
    const float f = x.x == -INFINITY ? 0.f : exp2f(x.x - top);
    total += f * x.y;  // NaN where the stretch's sum is, whatever f
#pragma unroll
    for (int e = 0; e < VEC; ++e) y[e] += f * p.e[e];
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) warp_sum_of[warp][lane * VEC + e] = y[e];
  if (lane == 0) warp_total[warp] = total;
  __syncthreads();
  total = (warp_total[0] + warp_total[1]) + (warp_total[2] + warp_total[3]);
  const long long to_row = out_index(L, b, h, row);
  if (threadIdx.x < D) {
    const int d = threadIdx.x;
    const float v = (warp_sum_of[0][d] + warp_sum_of[1][d]) + (warp_sum_of[2][d] + warp_sum_of[3][d]);
    static_cast<T*>(a.out)[to_row * D + d] = Elem<T>::from_f(total == 0.f ? 0.f : v / total);
  }
  if (a.lse && threadIdx.x == 0) a.lse[to_row] = total == 0.f ? -INFINITY : (top + log2f(total)) / kLog2e;
}

namespace {

int tiles_of_rows(int rows) { return rows <= 8 ? 1 : 2; }  // NT

int stage_bytes(int D) { return 2 * at_keys(D) * (D / 2 + D / kKv4Group * 4); }

size_t attn_smem(int D, int NT) {
  const size_t ring = static_cast<size_t>(kAtWarps) * at_stages(D) * stage_bytes(D);
  const size_t sums = static_cast<size_t>(kAtWarps) * 8 * NT * (D + 4) * sizeof(float);
  return std::max(ring, sums);
}

// Stretches for about eight CTAs an SM, of at least 128 places: two for every one that fits
// at head_dim 128 with up to 8 query rows a key head (24 x 6000 places of 8 heads: 62 us;
// with six CTAs an SM 70, with sixteen 69), 1.6 at head_dim 64, four with more rows, for
// which other counts were not measured. Sequences of up to 512 places stay whole: one launch
// instead of two (one sequence of 300: 8.8 -> 7.6 us on the GPU). The lengths lie on the
// device, so the page table's width stands for them: under a table much wider than its
// sequences the stretches are few and long (8 heads of 128, one sequence of 2000 places:
// 9.1 us, under a table of 131072 places 19.0; 8 of 4000 places: 22.6 and 67.2).
AttnLaunch plan(const Kv4AttnArgs& a) {
  AttnLaunch L{};
  L.a = a;
  L.group = a.Hq / a.c.heads;
  L.rows = a.T * L.group;
  const int NT = tiles_of_rows(L.rows);
  L.row_tiles = (L.rows + 8 * NT - 1) / (8 * NT);
  int nsm = 0;
  if (cached_sm_count(&nsm) != cudaSuccess) nsm = 148;
  const long long room = std::max(1LL, static_cast<long long>(a.max_pages) * a.c.page);
  const long long all = room * a.B * a.c.heads * L.row_tiles;
  const long long wish = room <= 512 ? room : all / (8LL * nsm) + 1;
  long long stretch = (std::min<long long>(wish, room) + 127) / 128 * 128;
  stretch = std::min<long long>(std::max<long long>(stretch, 128), kAtMaxStretch);
  L.stretch = static_cast<int>(stretch);
  L.q_packs = (reinterpret_cast<uintptr_t>(a.q) & 15u) == 0 && a.qs[0] % 8 == 0 && a.qs[1] % 8 == 0 && a.qs[2] % 8 == 0;
  L.splits = static_cast<int>((room + stretch - 1) / stretch);
  return L;
}

size_t parts(const AttnLaunch& L) {
  const int NT = tiles_of_rows(L.rows);
  return static_cast<size_t>(L.a.B) * L.a.c.heads * L.row_tiles * L.splits * 8 * NT;
}

template <typename T, int D, int NT>
cudaError_t attn_t(const AttnLaunch& L, cudaStream_t st) {
  const void* fn = reinterpret_cast<const void*>(&kv4_attn_kernel<T, D, NT>);
  const size_t smem = attn_smem(D, NT);
  cudaError_t e = ensure_dynamic_smem(fn, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  const dim3 grid(static_cast<unsigned>(L.splits) * L.row_tiles, L.a.c.heads, L.a.B);
  kv4_attn_kernel<T, D, NT><<<grid, kAtWarps * 32, smem, st>>>(L);
  if ((e = cudaGetLastError()) != cudaSuccess || L.splits == 1) return e;
  const long long rows = static_cast<long long>(L.a.B) * L.a.c.heads * L.rows;
  // a programmatic dependent: its launch overlaps the attention (3 us less a call)
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_join_kernel<T, D>, L, 8 * NT);
}

template <typename T>
cudaError_t attn_dt(const AttnLaunch& L, cudaStream_t st) {
  const int NT = tiles_of_rows(L.rows);
  if (L.a.c.D == 64) return NT == 1 ? attn_t<T, 64, 1>(L, st) : attn_t<T, 64, 2>(L, st);
  return NT == 1 ? attn_t<T, 128, 1>(L, st) : attn_t<T, 128, 2>(L, st);
}

}  // namespace

size_t kv4_attention_workspace_bytes(const Kv4AttnArgs& a) {
  const AttnLaunch L = plan(a);
  if (L.splits == 1) return 0;
  return parts(L) * (a.c.D + 2) * sizeof(float);
}

cudaError_t kv4_attention_launch(int dtype, const Kv4AttnArgs& a, cudaStream_t st) {
  AttnLaunch L = plan(a);
  if (static_cast<long long>(L.splits) * L.row_tiles > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  L.part_o = static_cast<float*>(a.workspace);
  L.part_ml = reinterpret_cast<float2*>(L.part_o + parts(L) * a.c.D);
  return dtype == ATTNRES_DTYPE_BF16 ? attn_dt<__nv_bfloat16>(L, st) : attn_dt<__half>(L, st);
}

cudaError_t read_kv4_attn_status(unsigned* status, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(status, g_kv4_attn_status, sizeof(unsigned));
  if (e != cudaSuccess || !reset) return e;
  const unsigned zero = 0;
  return cudaMemcpyToSymbol(g_kv4_attn_status, &zero, sizeof(unsigned));
}

}  // namespace attnres
