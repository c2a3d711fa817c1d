// Products of rows with the weights of the experts they were routed to, and their gradients.
//
//   rows:   z[slot, k, :] = W_e x[row(slot), k, :]        (or W_e^T g for the gradient in x)
//   weight: dW[e] = sum over e's rows of (w_slot g) x^T
//   join:   out[t, k, :] = sum_j w[t, j] z[(t, j), k, :], and the products <z, x> that the routing
//           weights' gradient needs, in slot order
//
// Bound by the tensor pipe for wide layers and many rows, by memory for narrow ones.  The rows of an
// expert (from the plan's order; all components of a slot next to each other) form tiles of 128 that
// meet BN of its outputs in one tcgen05.mma accumulator.  Producer warps gather the rows with 16-byte
// loads into 128-byte-swizzled shared memory slabs (64 two-byte elements a row), so that the same
// slab serves an operand whose rows are its M or N index (K-major) and one whose rows are the
// contraction index (MN-major: the gradient products read W and the rows untransposed).
//   32 bits: an element is the sum of three bfloat16 (8 + 8 + 8 significand bits); the six products
//   down to 2^-16 of the leading one are accumulated in fp32, the rest is below 2^-24.
//   8 bits: e4m3 operands, the row's and the output's scale multiply the accumulator.
#include <algorithm>

#include "common.cuh"
#include "num.cuh"
#include "tc_common.cuh"

namespace fsc {
namespace {

struct e4m3 {
  uint8_t b;
};

constexpr int kThreads = 288;  // 8 producer / epilogue warps, 1 MMA warp
constexpr int kProducers = 256;
constexpr int BM = 128;
constexpr int kSlabRow = 128;  // bytes

template <typename T>
constexpr int planes_of = sizeof(T) == 4 ? 3 : 1;
template <typename T>
constexpr int chunk_of = sizeof(T) == 1 ? 16 : 8;  // elements of one 16-byte shared memory chunk

struct LinearArgs {
  const void* x;         // gathered rows
  const void* w;         // weights (rows product) or the second gathered operand (weight product: x)
  const float* row_weight;  // per slot factor, or null
  const float* x_scale;  // 8 bits: per gathered row
  const float* w_scale;  // 8 bits: [experts][N]
  const int32_t* offsets;
  const int32_t* order;
  int32_t* status;
  void* out;
  int experts, per_token, comps;  // per_token: slots of a token
  int x_by_slot, w_by_slot;       // gathered operand has a row for each slot, not each token
  int N, Kd;                      // rows product: outputs, contraction; weight product: inputs I, outputs O in Kd
  int tiles_n;
  int splits;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t dst, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// x as the sum of three bfloat16: each is the rounded remainder of the ones before it.  Where the
// first would round past the largest finite value, the first two are cut instead (so that no partial
// sum passes it either); infinities and NaN have no rest.
__device__ __forceinline__ void split3(float x, uint16_t* p) {
  __nv_bfloat16 h = __float2bfloat16_rn(x);
  const bool cut = fabsf(__bfloat162float(h)) == INFINITY;
  if (cut) h = __ushort_as_bfloat16((uint16_t)(__float_as_uint(x) >> 16));
  const float hf = __bfloat162float(h);
  const float r = fabsf(hf) < INFINITY ? x - hf : 0.f;
  const __nv_bfloat16 m = cut ? __ushort_as_bfloat16((uint16_t)(__float_as_uint(r) >> 16)) : __float2bfloat16_rn(r);
  const __nv_bfloat16 l = __float2bfloat16_rn(r - __bfloat162float(m));
  p[0] = __bfloat16_as_ushort(h), p[1] = __bfloat16_as_ushort(m), p[2] = __bfloat16_as_ushort(l);
}

// One 16-byte chunk (chunk_of<T> elements of one row from column c) on its way to shared memory.
// VEC: rows start on 16 bytes and hold whole chunks' worth of 16-byte pieces.
template <typename T, bool VEC>
struct Piece {
  static constexpr int CE = chunk_of<T>;
  T v[CE];
  __device__ __forceinline__ void load(const T* row, int c, int cols) {
    if constexpr (VEC) {
      constexpr int E = 16 / sizeof(T);
#pragma unroll
      for (int b = 0; b < CE; b += E) {
        uint4 q = make_uint4(0, 0, 0, 0);
        if (row != nullptr && c + b < cols) q = __ldg(reinterpret_cast<const uint4*>(row + c + b));
        *reinterpret_cast<uint4*>(&v[b]) = q;
      }
    } else {
#pragma unroll
      for (int i = 0; i < CE; ++i) {
        if (row != nullptr && c + i < cols)
          v[i] = row[c + i];
        else
          memset(&v[i], 0, sizeof(T));
      }
    }
  }
  template <bool SCALED>
  __device__ __forceinline__ void store(uint32_t dst, uint32_t plane, float f) {
    if constexpr (sizeof(T) == 4) {
      alignas(16) uint16_t h[3][8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint16_t p[3];
        split3(SCALED ? v[i] * f : v[i], p);
        h[0][i] = p[0], h[1][i] = p[1], h[2][i] = p[2];
      }
#pragma unroll
      for (int q = 0; q < 3; ++q) st_shared16(dst + q * plane, *reinterpret_cast<uint4*>(h[q]));
    } else {
      if constexpr (SCALED) {  // one rounding of w g to the rows' type, as if g had been stored scaled
#pragma unroll
        for (int i = 0; i < CE; ++i) v[i] = from_f32<T>(to_f32(v[i]) * f);
      }
      st_shared16(dst, *reinterpret_cast<uint4*>(v));
    }
  }
};

// Byte offset of 16-byte chunk c (0..7) of row r in a 128-byte-swizzled slab.
__device__ __forceinline__ uint32_t slab_at(int r, int c) { return r * kSlabRow + ((c ^ (r & 7)) << 4); }

// Shared-memory matrix descriptor, 128-byte swizzle: `sbo` bytes between groups of eight slab rows;
// MN-major operands wider than 64 elements continue `lbo` bytes on.
__device__ __forceinline__ uint64_t desc128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)((lbo >> 4) & 0x3FFF) << 16 |
         (uint64_t)((sbo >> 4) & 0x3FFF) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

template <typename T>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (sizeof(T) == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
        "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
        "r"(accumulate)
        : "memory");
}

// Instruction descriptor: fp32 accumulator; f16 = 0 / bf16 = 1 (e4m3 = 0); bits 15 and 16: A and B MN-major.
template <typename T>
constexpr uint32_t idesc_of(int n, bool a_mn, bool b_mn) {
  constexpr uint32_t fmt = std::is_same<T, __half>::value || sizeof(T) == 1 ? 0 : 1;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}

// The products of planes (p of A, q of B) that count: 2^-8 apart each, kept while p + q <= 2.
template <typename T, int BN, bool A_MN, bool B_MN>
__device__ __forceinline__ void mma_stage(uint32_t tmem, uint32_t sa, uint32_t sb, bool first) {
  constexpr int P = planes_of<T>;
  constexpr uint32_t A_PLANE = BM * kSlabRow, B_PLANE = BN * kSlabRow;
  constexpr uint32_t A_STEP = A_MN ? 2048 : 32, B_STEP = B_MN ? 2048 : 32;
  constexpr uint32_t LBO = 64 * kSlabRow;  // 64 contraction rows of a slab
  constexpr uint32_t id = idesc_of<T>(BN, A_MN, B_MN);
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int q = 0; q < P; ++q)
        if (p + q < (P == 3 ? 3 : 1))
          mma_ss<T>(tmem, desc128(sa + p * A_PLANE + k * A_STEP, A_MN ? LBO : 16, 1024),
                    desc128(sb + q * B_PLANE + k * B_STEP, B_MN ? LBO : 16, 1024), id,
                    !(first && k == 0 && p == 0 && q == 0));
}

template <typename T, int BN>
struct Shape {
  static constexpr int P = planes_of<T>;
  static constexpr int A_BYTES = P * BM * kSlabRow, B_BYTES = P * BN * kSlabRow;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = P == 3 ? (BN == 64 ? 3 : 2) : (BN == 64 ? 4 : 3);  // 1 bits: two blocks per SM
  static constexpr int SMEM = STAGES * STAGE + 1024;
};

struct Barriers {
  uint64_t full[4], empty[4], done;
  uint32_t tmem;
  int32_t row[BM];   // gathered row of a tile row, -1: none
  int32_t slot[BM];
  int expert, first, rows;  // the expert, the tile's first row in it, the rows it has
};

// Finds the expert of row tile `tile` (tiles of BM rows, experts in order); warp 0 only.
__device__ __forceinline__ void find_tile(const LinearArgs& a, int tile, Barriers* s) {
  const int lane = threadIdx.x & 31;
  const int per = (a.experts + 31) / 32, lo = min(lane * per, a.experts), hi = min(lo + per, a.experts);
  int mine = 0;
  for (int e = lo; e < hi; ++e) mine += ((a.offsets[e + 1] - a.offsets[e]) * a.comps + BM - 1) / BM;
  int x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += t;
  }
  int start = x - mine;
  if (lane == 0) s->expert = -1;
  __syncwarp();
  if (tile >= start && tile < x) {
    for (int e = lo; e < hi; ++e) {
      const int rows = (a.offsets[e + 1] - a.offsets[e]) * a.comps, n = (rows + BM - 1) / BM;
      if (tile < start + n) {
        s->expert = e, s->first = (tile - start) * BM, s->rows = rows;
        break;
      }
      start += n;
    }
  }
}

__device__ __forceinline__ int gathered_row(const LinearArgs& a, int by_slot, int slot, int comp) {
  return (by_slot ? slot : slot / a.per_token) * a.comps + comp;
}

template <bool ASYNC>
struct Arrival {
  static constexpr int LAG = ASYNC ? 1 : 0;
  // Stage `kc` has been written (or its copies issued): publishes the stage LAG behind it.
  __device__ static __forceinline__ void publish(Barriers* s, int kc, int stages) {
    if constexpr (ASYNC) {
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (kc < LAG) return;
      asm volatile("cp.async.wait_group %0;" ::"n"(LAG) : "memory");
      kc -= LAG;
    }
    fence_async_shared();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) tc::mbar_arrive(&s->full[kc % stages]);
  }
  __device__ static __forceinline__ void finish(Barriers* s, int nk, int stages) {
    if constexpr (ASYNC) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_async_shared();
      __syncwarp();
      if ((threadIdx.x & 31) == 0 && nk > 0) tc::mbar_arrive(&s->full[(nk - 1) % stages]);
    }
  }
};

__device__ __forceinline__ void pipeline_init(Barriers* s, int stages, uint32_t cols) {
  if (threadIdx.x == kProducers) {
    for (int i = 0; i < stages; ++i) tc::mbar_init(&s->full[i], kProducers / 32), tc::mbar_init(&s->empty[i], 1);
    tc::mbar_init(&s->done, 1);
    tc::fence_mbar_init();
  }
  if (threadIdx.x >= kProducers) {
    __syncwarp();
    tc::tmem_alloc(&s->tmem, cols);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
}

template <typename T, int BN, bool A_MN, bool B_MN>
__device__ __forceinline__ void mma_warp(const LinearArgs& a, Barriers* s, uint32_t base, int nk) {
  using S = Shape<T, BN>;
  if (threadIdx.x == kProducers) {
    bool ok = true;
    for (int kc = 0; kc < nk && ok; ++kc) {
      const int st = kc % S::STAGES;
      ok = tc::mbar_wait(&s->full[st], (kc / S::STAGES) & 1, a.status, 1);
      if (!ok) break;
      tc::tc_fence_after();
      mma_stage<T, BN, A_MN, B_MN>(s->tmem, base + st * S::STAGE, base + st * S::STAGE + S::A_BYTES, kc == 0);
      tc::mma_commit(&s->empty[st]);
    }
    tc::mma_commit(&s->done);
  }
  __syncwarp();
}

// ---- rows product --------------------------------------------------------------------------------
// OUT float: unscaled products in slot order for the join; else rows of the output's type, times the
// slot's weight.  B_MN: the weights' rows are the contraction index (W^T).
template <typename T, typename OUT, int BN, bool B_MN, bool VEC>
__global__ void __launch_bounds__(kThreads) rows_kernel(LinearArgs a) {
  using S = Shape<T, BN>;
  constexpr int CE = chunk_of<T>, KC = 8 * CE;
  constexpr bool ASYNC = VEC && sizeof(T) != 4;
  extern __shared__ uint8_t dyn[];
  __shared__ Barriers s;
  const uint32_t base = (tc::smem_u32(dyn) + 1023) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 0) find_tile(a, blockIdx.x / a.tiles_n, &s);
  __syncthreads();
  if (s.expert < 0) return;  // beyond the last tile
  const int e = s.expert, n0 = (blockIdx.x % a.tiles_n) * BN;
  if (tid < BM) {
    const int r = s.first + tid;
    int row = -1, slot = -1;
    if (r < s.rows) {
      slot = a.order[a.offsets[e] + r / a.comps];
      const int comp = r % a.comps;
      row = gathered_row(a, a.x_by_slot, slot, comp);
    }
    s.row[tid] = row;
    s.slot[tid] = slot;
  }
  pipeline_init(&s, S::STAGES, BN);
  const int nk = (a.Kd + KC - 1) / KC;
  const T* x = static_cast<const T*>(a.x);
  const T* w = static_cast<const T*>(a.w) + (int64_t)e * a.N * a.Kd;
  if (warp < 8) {
    bool ok = true;
    constexpr int NA = BM * 8 / kProducers, NB = BN * 8 / kProducers;
    for (int kc = 0; kc < nk; ++kc) {
      const int st = kc % S::STAGES;
      const uint32_t sa = base + st * S::STAGE, sb = sa + S::A_BYTES;
      auto a_row = [&](int i) -> const T* {
        const int row = s.row[(tid + i * kProducers) >> 3];
        return row >= 0 ? x + (int64_t)row * a.Kd : nullptr;
      };
      auto b_row = [&](int i) -> const T* {
        const int q = tid + i * kProducers;
        if constexpr (B_MN) {
          const int k = kc * KC + q / (BN / 8);
          return k < a.Kd ? w + (int64_t)k * a.N : nullptr;
        } else {
          const int n = n0 + (q >> 3);
          return n < a.N ? w + (int64_t)n * a.Kd : nullptr;
        }
      };
      auto a_dst = [&](int i) {
        const int q = tid + i * kProducers;
        return sa + slab_at(q >> 3, q & 7);
      };
      auto b_dst = [&](int i) {
        const int q = tid + i * kProducers;
        if constexpr (B_MN) {
          const int k = q / (BN / 8), c = q % (BN / 8);
          return sb + (c >> 3) * (64 * kSlabRow) + slab_at(k, c & 7);
        } else {
          return sb + slab_at(q >> 3, q & 7);
        }
      };
      auto b_col = [&](int i) {
        const int q = tid + i * kProducers;
        return B_MN ? n0 + (q % (BN / 8)) * CE : kc * KC + (q & 7) * CE;
      };
      const int b_cols = B_MN ? a.N : a.Kd;
      const int a_col = kc * KC + (tid & 7) * CE;
      if constexpr (ASYNC) {
        if (kc >= S::STAGES) ok = ok && tc::mbar_wait(&s.empty[st], (kc / S::STAGES - 1) & 1, a.status, 2);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < NA; ++i) {
          const T* r = a_row(i);
          const bool in = r != nullptr && a_col < a.Kd;
          cp_async16(a_dst(i), in ? r + a_col : x, in);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          const T* r = b_row(i);
          const bool in = r != nullptr && b_col(i) < b_cols;
          cp_async16(b_dst(i), in ? r + b_col(i) : w, in);
        }
      } else {
        Piece<T, VEC> pa[NA], pb[NB];
#pragma unroll
        for (int i = 0; i < NA; ++i) pa[i].load(a_row(i), a_col, a.Kd);
#pragma unroll
        for (int i = 0; i < NB; ++i) pb[i].load(b_row(i), b_col(i), b_cols);
        if (kc >= S::STAGES) ok = ok && tc::mbar_wait(&s.empty[st], (kc / S::STAGES - 1) & 1, a.status, 2);
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < NA; ++i) pa[i].template store<false>(a_dst(i), BM * kSlabRow, 1.f);
#pragma unroll
        for (int i = 0; i < NB; ++i) pb[i].template store<false>(b_dst(i), BN * kSlabRow, 1.f);
      }
      Arrival<ASYNC>::publish(&s, kc, S::STAGES);
    }
    Arrival<ASYNC>::finish(&s, ok ? nk : 0, S::STAGES);
    ok = tc::mbar_wait(&s.done, 0, a.status, 3) && ok;
    tc::tc_fence_after();
    const int m = (warp & 3) * 32 + lane, slot = s.slot[m];
    float f = 1.f;
    if (slot >= 0 && a.row_weight) f = a.row_weight[slot];
    if constexpr (sizeof(T) == 1)
      if (slot >= 0) f *= a.x_scale[a.x_by_slot ? slot : slot / a.per_token];
    OUT* out = static_cast<OUT*>(a.out);
    if (slot >= 0) out += ((int64_t)slot * a.comps + (s.first + m) % a.comps) * a.N;
    const bool wide = a.N % (16 / sizeof(OUT)) == 0;
#pragma unroll
    for (int cb = 0; cb < BN / 64; ++cb) {
      const int c0 = (warp >> 2) * (BN / 2) + cb * 32;
      uint32_t v[32];
      __syncwarp();
      tc::tmem_ld32(s.tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0, v);
      tc::tmem_wait_ld();
      if (slot < 0 || !ok) continue;
      constexpr int E = 16 / sizeof(OUT);
#pragma unroll
      for (int j = 0; j < 32; j += E) {
        const int n = n0 + c0 + j;
        Pack<OUT, E> p;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          float y = __uint_as_float(v[j + i]) * f;
          if constexpr (sizeof(T) == 1) y *= n + i < a.N ? a.w_scale[(int64_t)e * a.N + n + i] : 0.f;
          p.v[i] = from_f32<OUT>(y);
        }
        if (wide) {
          if (n < a.N) *reinterpret_cast<Pack<OUT, E>*>(out + n) = p;
        } else {
#pragma unroll
          for (int i = 0; i < E; ++i)
            if (n + i < a.N) out[n + i] = p.v[i];
        }
      }
    }
    tc::tc_fence_before();
  } else {
    mma_warp<T, BN, false, B_MN>(a, &s, base, nk);
  }
  __syncthreads();
  if (warp == 8) {
    tc::tc_fence_after();
    tc::tmem_dealloc(s.tmem, BN);
  }
}

// ---- weight product ------------------------------------------------------------------------------
// dW[e][o][i]: both operands gathered, the rows are the contraction index.  Kd: O, N: I.
template <typename T, typename OUT, int BN, bool VEC>
__global__ void __launch_bounds__(kThreads) weight_kernel(LinearArgs a) {
  using S = Shape<T, BN>;
  constexpr int CE = 8, KC = 64;
  extern __shared__ uint8_t dyn[];
  __shared__ Barriers s;
  const uint32_t base = (tc::smem_u32(dyn) + 1023) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int b = blockIdx.x;
  const int split = b % a.splits;
  b /= a.splits;
  const int n0 = (b % a.tiles_n) * BN;
  b /= a.tiles_n;
  const int tiles_m = (a.Kd + BM - 1) / BM;
  const int m0 = (b % tiles_m) * BM, e = b / tiles_m;
  const int rows = (a.offsets[e + 1] - a.offsets[e]) * a.comps;
  const int part = ((rows + a.splits - 1) / a.splits + KC - 1) / KC * KC;
  const int lo = min(split * part, rows), hi = min(lo + part, rows);
  const int nk = (hi - lo + KC - 1) / KC;
  pipeline_init(&s, S::STAGES, BN);
  const T* g = static_cast<const T*>(a.x);
  const T* x = static_cast<const T*>(a.w);
  const int32_t* order = a.order + a.offsets[e];
  if (warp < 8) {
    bool ok = true;
    constexpr int NA = BM * 8 / kProducers, NB = BN * 8 / kProducers;
    for (int kc = 0; kc < nk; ++kc) {
      const int st = kc % S::STAGES;
      const uint32_t sa = base + st * S::STAGE, sb = sa + S::A_BYTES;
      Piece<T, VEC> pa[NA], pb[NB];
      float f[NA];
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        const int q = tid + i * kProducers, r = lo + kc * KC + q / (BM / 8);
        const T* row = nullptr;
        f[i] = 1.f;
        if (r < hi) {
          const int slot = order[r / a.comps];
          row = g + (int64_t)gathered_row(a, a.x_by_slot, slot, r % a.comps) * a.Kd;
          if (a.row_weight) f[i] = a.row_weight[slot];
        }
        pa[i].load(row, m0 + (q % (BM / 8)) * CE, a.Kd);
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int q = tid + i * kProducers, r = lo + kc * KC + q / (BN / 8);
        const T* row = nullptr;
        if (r < hi) row = x + (int64_t)gathered_row(a, a.w_by_slot, order[r / a.comps], r % a.comps) * a.N;
        pb[i].load(row, n0 + (q % (BN / 8)) * CE, a.N);
      }
      if (kc >= S::STAGES) ok = ok && tc::mbar_wait(&s.empty[st], (kc / S::STAGES - 1) & 1, a.status, 2);
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        const int q = tid + i * kProducers, k = q / (BM / 8), c = q % (BM / 8);
        const uint32_t dst = sa + (c >> 3) * (64 * kSlabRow) + slab_at(k, c & 7);
        if (a.row_weight)
          pa[i].template store<true>(dst, BM * kSlabRow, f[i]);
        else
          pa[i].template store<false>(dst, BM * kSlabRow, 1.f);
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int q = tid + i * kProducers, k = q / (BN / 8), c = q % (BN / 8);
        pb[i].template store<false>(sb + (c >> 3) * (64 * kSlabRow) + slab_at(k, c & 7), BN * kSlabRow, 1.f);
      }
      Arrival<false>::publish(&s, kc, S::STAGES);
    }
    ok = tc::mbar_wait(&s.done, 0, a.status, 3) && ok;
    tc::tc_fence_after();
    const int o = m0 + (warp & 3) * 32 + lane;
    OUT* out = static_cast<OUT*>(a.out) + (((int64_t)split * a.experts + e) * a.Kd + min(o, a.Kd - 1)) * a.N;
    const bool wide = a.N % (16 / sizeof(OUT)) == 0;
#pragma unroll
    for (int cb = 0; cb < BN / 64; ++cb) {
      const int c0 = (warp >> 2) * (BN / 2) + cb * 32;
      uint32_t v[32];
      __syncwarp();
      if (nk > 0) {
        tc::tmem_ld32(s.tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0, v);
        tc::tmem_wait_ld();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0;
      }
      if (o >= a.Kd || !ok) continue;
      constexpr int E = 16 / sizeof(OUT);
#pragma unroll
      for (int j = 0; j < 32; j += E) {
        const int n = n0 + c0 + j;
        Pack<OUT, E> p;
#pragma unroll
        for (int i = 0; i < E; ++i) p.v[i] = from_f32<OUT>(__uint_as_float(v[j + i]));
        if (wide) {
          if (n < a.N) *reinterpret_cast<Pack<OUT, E>*>(out + n) = p;
        } else {
#pragma unroll
          for (int i = 0; i < E; ++i)
            if (n + i < a.N) out[n + i] = p.v[i];
        }
      }
    }
    tc::tc_fence_before();
  } else {
    mma_warp<T, BN, true, true>(a, &s, base, nk);
  }
  __syncthreads();
  if (warp == 8) {
    tc::tc_fence_after();
    tc::tmem_dealloc(s.tmem, BN);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) split_sum_kernel(const float* part, int splits, int64_t n, T* out) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float s = part[i];
    for (int p = 1; p < splits; ++p) s += part[p * n + i];
    out[i] = from_f32<T>(s);
  }
}

// ---- join ----------------------------------------------------------------------------------------
struct JoinArgs {
  const float* z;         // [tokens * per_token][width]
  const int32_t* indices; // [tokens * per_token]
  const float* weights;   // per slot, or null: 1
  const void* x;          // rows to multiply z with, or null
  int x_by_slot;
  void* out;              // [tokens][width] sums, or null
  void* slot_out;         // [tokens * per_token][width] w z, or null
  float* dots;            // [tokens * per_token] <z, x>, or null
  int64_t tokens;
  int per_token, experts;
  int64_t width;
};

// NW warps share a token; each thread keeps the products of the S slots of a pass.
template <typename T, int NW, int S, int VE>
__global__ void __launch_bounds__(128) join_kernel(JoinArgs a) {
  constexpr int TPT = NW * 32;
  __shared__ float part[4][32];
  const int t = threadIdx.x % TPT;
  const int64_t token = (int64_t)blockIdx.x * (128 / TPT) + threadIdx.x / TPT;
  if (token >= a.tokens) return;
  for (int j0 = 0; j0 < a.per_token; j0 += S) {  // one pass unless a token has more than 32 slots
    float dot[S];
#pragma unroll
    for (int j = 0; j < S; ++j) dot[j] = 0.f;
    for (int64_t c = (int64_t)t * VE; c < a.width; c += TPT * VE) {
      float sum[VE], xs[VE];
#pragma unroll
      for (int i = 0; i < VE; ++i) sum[i] = 0.f, xs[i] = 0.f;
      if (a.x && !a.x_by_slot) {
        const Pack<T, VE> p = *reinterpret_cast<const Pack<T, VE>*>(static_cast<const T*>(a.x) + token * a.width + c);
#pragma unroll
        for (int i = 0; i < VE; ++i) xs[i] = to_f32(p.v[i]);
      }
#pragma unroll
      for (int j = 0; j < S; ++j) {
        if (j0 + j >= a.per_token) continue;
        const int64_t slot = token * a.per_token + j0 + j;
        const int e = a.indices[slot];
        const bool live = e >= 0 && e < a.experts;
        float z[VE];
        if (live) {
          constexpr int N = VE > 4 ? 4 : VE;
#pragma unroll
          for (int b = 0; b < VE; b += N) {
            const Pack<float, N> p = *reinterpret_cast<const Pack<float, N>*>(a.z + slot * a.width + c + b);
#pragma unroll
            for (int i = 0; i < N; ++i) z[b + i] = p.v[i];
          }
          if (a.x) {
            if (a.x_by_slot) {
              const Pack<T, VE> p =
                  *reinterpret_cast<const Pack<T, VE>*>(static_cast<const T*>(a.x) + slot * a.width + c);
#pragma unroll
              for (int i = 0; i < VE; ++i) xs[i] = to_f32(p.v[i]);
            }
#pragma unroll
            for (int i = 0; i < VE; ++i) dot[j] = fmaf(z[i], xs[i], dot[j]);
          }
        }
        const float f = live ? (a.weights ? a.weights[slot] : 1.f) : 0.f;
        if (a.slot_out) {
          Pack<T, VE> p;
#pragma unroll
          for (int i = 0; i < VE; ++i) p.v[i] = from_f32<T>(live ? z[i] * f : 0.f);
          *reinterpret_cast<Pack<T, VE>*>(static_cast<T*>(a.slot_out) + slot * a.width + c) = p;
        }
        if (live) {
#pragma unroll
          for (int i = 0; i < VE; ++i) sum[i] = fmaf(z[i], f, sum[i]);
        }
      }
      if (a.out) {
        Pack<T, VE> p;
#pragma unroll
        for (int i = 0; i < VE; ++i) p.v[i] = from_f32<T>(sum[i]);
        *reinterpret_cast<Pack<T, VE>*>(static_cast<T*>(a.out) + token * a.width + c) = p;
      }
    }
    if (a.dots) {
#pragma unroll
      for (int j = 0; j < S; ++j) {
        dot[j] = warp_sum(dot[j]);
        if (NW > 1 && (threadIdx.x & 31) == 0) part[threadIdx.x >> 5][j] = dot[j];
      }
      if (NW > 1) __syncthreads();
#pragma unroll
      for (int j = 0; j < S; ++j) {
        if (j0 + j < a.per_token && t == 0) {
          float d = dot[j];
          if (NW > 1) d = (part[0][j] + part[1][j]) + (part[2][j] + part[3][j]);
          a.dots[token * a.per_token + j0 + j] = d;
        }
      }
    }
  }
}

template <typename T, int NW, int VE>
int launch_join_s(const JoinArgs& a, cudaStream_t st) {
  const unsigned blocks = (unsigned)ceil_div(a.tokens, NW == 1 ? 4 : 1);
  if (a.per_token <= 2)
    join_kernel<T, NW, 2, VE><<<blocks, 128, 0, st>>>(a);
  else if (a.per_token <= 8)
    join_kernel<T, NW, 8, VE><<<blocks, 128, 0, st>>>(a);
  else
    join_kernel<T, NW, 32, VE><<<blocks, 128, 0, st>>>(a);
  return check_launch("expert_linear join");
}

template <typename T>
int launch_join(const JoinArgs& a, cudaStream_t st) {
  if (a.tokens == 0) return FSC_OK;
  constexpr int VE = 16 / sizeof(T);
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vec = a.width % VE == 0 && al(a.x) && al(a.out) && al(a.slot_out) && al(a.z);
  const bool block = a.width >= 1024;  // four warps a token where each still has 8 vectors or more
  if (vec) return block ? launch_join_s<T, 4, VE>(a, st) : launch_join_s<T, 1, VE>(a, st);
  return block ? launch_join_s<T, 4, 1>(a, st) : launch_join_s<T, 1, 1>(a, st);
}

// Zero rows for slots that no expert takes, where the product writes its output directly.
template <typename T>
__global__ void __launch_bounds__(256) zero_slots_kernel(const int32_t* indices, int experts, int64_t slots,
                                                         int64_t width, T* out) {
  for (int64_t s = blockIdx.x; s < slots; s += gridDim.x) {
    const int e = indices[s];
    if (e >= 0 && e < experts) continue;
    for (int64_t c = threadIdx.x; c < width; c += 256) out[s * width + c] = from_f32<T>(0.f);
  }
}

// ---- launches ------------------------------------------------------------------------------------
template <typename K>
int set_smem(K kernel, int bytes) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return check_launch("expert_linear");
  return FSC_OK;
}

template <typename T, typename OUT, int BN, bool B_MN, bool VEC>
int launch_rows4(const LinearArgs& a, int64_t row_tiles, cudaStream_t st) {
  auto k = rows_kernel<T, OUT, BN, B_MN, VEC>;
  FSC_TRY(set_smem(k, Shape<T, BN>::SMEM));
  k<<<(unsigned)(row_tiles * a.tiles_n), kThreads, Shape<T, BN>::SMEM, st>>>(a);
  return check_launch("expert_linear rows");
}

template <typename T, typename OUT, bool B_MN>
int launch_rows(LinearArgs a, int64_t slots, bool vec, cudaStream_t st) {
  const int bn = a.N <= 64 ? 64 : 128;
  a.tiles_n = (int)ceil_div(a.N, bn);
  const int64_t tiles = ceil_div(slots * a.comps, BM) + std::min<int64_t>(a.experts, slots);
  FSC_REQUIRE(tiles * a.tiles_n < (1ll << 31), "expert_linear: too many tiles");
  if (bn == 64)
    return vec ? launch_rows4<T, OUT, 64, B_MN, true>(a, tiles, st) : launch_rows4<T, OUT, 64, B_MN, false>(a, tiles, st);
  return vec ? launch_rows4<T, OUT, 128, B_MN, true>(a, tiles, st) : launch_rows4<T, OUT, 128, B_MN, false>(a, tiles, st);
}

template <typename T, typename OUT>
int launch_weight(LinearArgs a, bool vec, cudaStream_t st) {
  const int bn = a.N <= 64 ? 64 : 128;
  a.tiles_n = (int)ceil_div(a.N, bn);
  const int64_t blocks = (int64_t)a.experts * ceil_div(a.Kd, BM) * a.tiles_n * a.splits;
  FSC_REQUIRE(blocks < (1ll << 31), "expert_linear: too many tiles");
  auto go = [&](auto kernel, int smem) {
    FSC_TRY(set_smem(kernel, smem));
    kernel<<<(unsigned)blocks, kThreads, smem, st>>>(a);
    return check_launch("expert_linear weight gradient");
  };
  if (bn == 64)
    return vec ? go(weight_kernel<T, OUT, 64, true>, Shape<T, 64>::SMEM) : go(weight_kernel<T, OUT, 64, false>, Shape<T, 64>::SMEM);
  return vec ? go(weight_kernel<T, OUT, 128, true>, Shape<T, 128>::SMEM) : go(weight_kernel<T, OUT, 128, false>, Shape<T, 128>::SMEM);
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Parts into which an expert's rows are cut for its weight gradient: enough blocks for two per SM,
// and 1024 rows or more in a part.
int weight_splits(int64_t slots, int64_t comps, int64_t experts, int64_t outputs, int64_t inputs) {
  const int64_t tiles = experts * ceil_div(outputs, BM) * ceil_div(inputs, inputs <= 64 ? 64 : 128);
  const int64_t most = std::max<int64_t>(1, slots * comps / experts / 1024);
  return (int)std::max<int64_t>(1, std::min<int64_t>({ceil_div(296, tiles), most, 64}));
}

struct Sizes {
  int64_t tokens, per_token, comps, experts, inputs, outputs;
};

int check_sizes(const Sizes& z) {
  FSC_REQUIRE(z.tokens >= 0 && z.tokens < (1ll << 31) && z.per_token >= 1 && z.per_token <= 32 && z.comps >= 1 && z.comps <= 1024,
              "expert_linear: 1 to 32 slots a token, 1 to 1024 components");
  FSC_REQUIRE(z.experts >= 1 && z.experts <= 1024, "expert_linear: 1 to 1024 experts");
  FSC_REQUIRE(z.inputs >= 1 && z.inputs <= (1 << 20) && z.outputs >= 1 && z.outputs <= (1 << 20),
              "expert_linear: inputs and outputs must be between 1 and 2^20");
  FSC_REQUIRE(z.tokens * z.per_token * z.comps < (1ll << 31) - 256, "expert_linear: too many rows");
  return FSC_OK;
}

template <typename T, typename OUT>
int forward(const Sizes& z, LinearArgs a, const int32_t* indices, const float* weights, void* out, float* ws,
            cudaStream_t st) {
  const int64_t slots = z.tokens * z.per_token;
  constexpr int E = 16 / sizeof(T);
  const bool vec = z.inputs % E == 0 && al16(a.x) && al16(a.w);
  a.N = (int)z.outputs, a.Kd = (int)z.inputs;
  if (weights == nullptr || z.per_token == 1) {  // a row of the output for each product: written directly
    a.out = out, a.row_weight = weights;
    zero_slots_kernel<OUT><<<(unsigned)std::min<int64_t>(slots, 148 * 8), 256, 0, st>>>(
        indices, a.experts, slots, z.comps * z.outputs, static_cast<OUT*>(out));
    FSC_TRY(check_launch("expert_linear"));
    return launch_rows<T, OUT, false>(a, slots, vec, st);
  }
  a.out = ws;
  FSC_TRY((launch_rows<T, float, false>(a, slots, vec, st)));
  JoinArgs j{};
  j.z = ws, j.indices = indices, j.weights = weights, j.out = out;
  j.tokens = z.tokens, j.per_token = a.per_token, j.experts = a.experts, j.width = z.comps * z.outputs;
  return launch_join<OUT>(j, st);
}

template <typename T>
int backward(const Sizes& z, LinearArgs a, const void* grad_out, const void* x, const void* w, const int32_t* indices,
             const float* weights, int slots_in, void* grad_x, void* grad_w, float* grad_weights, char* ws,
             cudaStream_t st) {
  const int64_t slots = z.tokens * z.per_token;
  constexpr int E = 16 / sizeof(T);
  const bool vec = z.inputs % E == 0 && z.outputs % E == 0 && al16(grad_out) && al16(x) && al16(w);
  const int out_by_slot = weights == nullptr;
  if (grad_x || grad_weights) {
    LinearArgs r = a;
    r.x = grad_out, r.w = w, r.N = (int)z.inputs, r.Kd = (int)z.outputs, r.x_by_slot = out_by_slot, r.row_weight = nullptr;
    r.out = ws;
    FSC_TRY((launch_rows<T, float, true>(r, slots, vec, st)));
    JoinArgs j{};
    j.z = reinterpret_cast<float*>(ws), j.indices = indices, j.weights = weights;
    j.tokens = z.tokens, j.per_token = a.per_token, j.experts = a.experts, j.width = z.comps * z.inputs;
    j.x = grad_weights ? x : nullptr, j.x_by_slot = slots_in, j.dots = grad_weights;
    (slots_in ? j.slot_out : j.out) = grad_x;
    FSC_TRY(launch_join<T>(j, st));
    ws += ((size_t)slots * z.comps * z.inputs * 4 + 255) & ~size_t(255);
  }
  if (grad_w) {
    LinearArgs g = a;
    g.x = grad_out, g.w = x, g.row_weight = weights, g.x_by_slot = out_by_slot, g.w_by_slot = slots_in;
    g.N = (int)z.inputs, g.Kd = (int)z.outputs;
    g.splits = weight_splits(slots, z.comps, z.experts, z.outputs, z.inputs);
    if (g.splits == 1) {
      g.out = grad_w;
      return launch_weight<T, T>(g, vec, st);
    }
    g.out = ws;
    FSC_TRY((launch_weight<T, float>(g, vec, st)));
    const int64_t n = z.experts * z.outputs * z.inputs;
    split_sum_kernel<T><<<(unsigned)std::min<int64_t>(ceil_div(n, 256), 148 * 8), 256, 0, st>>>(
        reinterpret_cast<float*>(ws), g.splits, n, static_cast<T*>(grad_w));
    return check_launch("expert_linear weight gradient");
  }
  return FSC_OK;
}

}  // namespace
}  // namespace fsc

using namespace fsc;

extern "C" {

size_t fsc_expert_linear_workspace_bytes(int64_t tokens, int64_t per_token, int64_t comps, int64_t experts,
                                         int64_t inputs, int64_t outputs, int weighted) {
  const Sizes z{tokens, per_token, comps, experts, inputs, outputs};
  if (check_sizes(z) != FSC_OK || !weighted || per_token == 1) return 0;
  return (size_t)(tokens * per_token * comps) * (size_t)outputs * sizeof(float);
}

int fsc_expert_linear(int dtype, const void* x, const void* w, const int32_t* indices, const float* weights,
                      const int32_t* offsets, const int32_t* order, int32_t* status, void* out, int64_t tokens,
                      int64_t per_token, int64_t comps, int64_t experts, int64_t inputs, int64_t outputs,
                      int x_by_slot, void* workspace, size_t workspace_bytes, void* stream) {
  const Sizes z{tokens, per_token, comps, experts, inputs, outputs};
  FSC_REQUIRE(dtype == FSC_F32 || dtype == FSC_BF16 || dtype == FSC_F16, "expert_linear: dtype must be f32, bf16 or f16");
  FSC_TRY(check_sizes(z));
  if (tokens == 0) return FSC_OK;
  FSC_REQUIRE(x && w && indices && offsets && order && status && out, "expert_linear: null pointer");
  FSC_REQUIRE(workspace_bytes >= fsc_expert_linear_workspace_bytes(tokens, per_token, comps, experts, inputs, outputs,
                                                                   weights != nullptr),
              "expert_linear: workspace too small");
  LinearArgs a{};
  a.x = x, a.w = w, a.offsets = offsets, a.order = order, a.status = status;
  a.experts = (int)experts, a.per_token = (int)per_token, a.comps = (int)comps, a.x_by_slot = x_by_slot != 0;
  float* ws = static_cast<float*>(workspace);
  cudaStream_t st = as_stream(stream);
  if (dtype == FSC_F32) return forward<float, float>(z, a, indices, weights, out, ws, st);
  if (dtype == FSC_BF16) return forward<__nv_bfloat16, __nv_bfloat16>(z, a, indices, weights, out, ws, st);
  return forward<__half, __half>(z, a, indices, weights, out, ws, st);
}

int fsc_expert_linear_q8(int out_dtype, const void* x, const float* x_scale, const void* w, const float* w_scale,
                         const int32_t* indices, const float* weights, const int32_t* offsets, const int32_t* order,
                         int32_t* status, void* out, int64_t tokens, int64_t per_token, int64_t comps,
                         int64_t experts, int64_t inputs, int64_t outputs, int x_by_slot, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const Sizes z{tokens, per_token, comps, experts, inputs, outputs};
  FSC_REQUIRE(out_dtype == FSC_F32 || out_dtype == FSC_BF16 || out_dtype == FSC_F16,
              "expert_linear_q8: out_dtype must be f32, bf16 or f16");
  FSC_REQUIRE(comps == 1, "expert_linear_q8: rows have one component");
  FSC_TRY(check_sizes(z));
  if (tokens == 0) return FSC_OK;
  FSC_REQUIRE(x && x_scale && w && w_scale && indices && offsets && order && status && out,
              "expert_linear_q8: null pointer");
  FSC_REQUIRE(workspace_bytes >= fsc_expert_linear_workspace_bytes(tokens, per_token, comps, experts, inputs, outputs,
                                                                   weights != nullptr),
              "expert_linear_q8: workspace too small");
  LinearArgs a{};
  a.x = x, a.w = w, a.x_scale = x_scale, a.w_scale = w_scale, a.offsets = offsets, a.order = order, a.status = status;
  a.experts = (int)experts, a.per_token = (int)per_token, a.comps = 1, a.x_by_slot = x_by_slot != 0;
  float* ws = static_cast<float*>(workspace);
  cudaStream_t st = as_stream(stream);
  if (out_dtype == FSC_F32) return forward<e4m3, float>(z, a, indices, weights, out, ws, st);
  if (out_dtype == FSC_BF16) return forward<e4m3, __nv_bfloat16>(z, a, indices, weights, out, ws, st);
  return forward<e4m3, __half>(z, a, indices, weights, out, ws, st);
}

size_t fsc_expert_linear_backward_workspace_bytes(int64_t tokens, int64_t per_token, int64_t comps, int64_t experts,
                                                  int64_t inputs, int64_t outputs, int weight_gradient) {
  const Sizes z{tokens, per_token, comps, experts, inputs, outputs};
  if (check_sizes(z) != FSC_OK) return 0;
  size_t n = ((size_t)(tokens * per_token * comps) * (size_t)inputs * sizeof(float) + 255) & ~size_t(255);
  const int splits = weight_splits(tokens * per_token, comps, experts, outputs, inputs);
  if (weight_gradient && splits > 1) n += (size_t)splits * (size_t)(experts * outputs) * (size_t)inputs * sizeof(float);
  return n;
}

int fsc_expert_linear_backward(int dtype, const void* grad_out, const void* x, const void* w, const int32_t* indices,
                               const float* weights, const int32_t* offsets, const int32_t* order, int32_t* status,
                               void* grad_x, void* grad_w, float* grad_weights, int64_t tokens, int64_t per_token,
                               int64_t comps, int64_t experts, int64_t inputs, int64_t outputs, int x_by_slot,
                               void* workspace, size_t workspace_bytes, void* stream) {
  const Sizes z{tokens, per_token, comps, experts, inputs, outputs};
  FSC_REQUIRE(dtype == FSC_F32 || dtype == FSC_BF16 || dtype == FSC_F16,
              "expert_linear_backward: dtype must be f32, bf16 or f16");
  FSC_TRY(check_sizes(z));
  cudaStream_t st = as_stream(stream);
  if (tokens == 0) {
    const size_t n = (size_t)(experts * outputs) * (size_t)inputs * (dtype == FSC_F32 ? 4 : 2);
    if (grad_w && cudaMemsetAsync(grad_w, 0, n, st) != cudaSuccess) return check_launch("expert_linear_backward");
    return FSC_OK;
  }
  FSC_REQUIRE(grad_out && x && w && indices && offsets && order && status, "expert_linear_backward: null pointer");
  FSC_REQUIRE(!grad_weights || weights, "expert_linear_backward: grad_weights needs weights");
  FSC_REQUIRE(workspace && workspace_bytes >= fsc_expert_linear_backward_workspace_bytes(
                                                 tokens, per_token, comps, experts, inputs, outputs, grad_w != nullptr),
              "expert_linear_backward: workspace too small");
  LinearArgs a{};
  a.offsets = offsets, a.order = order, a.status = status;
  a.experts = (int)experts, a.per_token = (int)per_token, a.comps = (int)comps;
  char* ws = static_cast<char*>(workspace);
  if (dtype == FSC_F32)
    return backward<float>(z, a, grad_out, x, w, indices, weights, x_by_slot != 0, grad_x, grad_w, grad_weights, ws, st);
  if (dtype == FSC_BF16)
    return backward<__nv_bfloat16>(z, a, grad_out, x, w, indices, weights, x_by_slot != 0, grad_x, grad_w, grad_weights,
                                   ws, st);
  return backward<__half>(z, a, grad_out, x, w, indices, weights, x_by_slot != 0, grad_x, grad_w, grad_weights, ws, st);
}

}  // extern "C"
