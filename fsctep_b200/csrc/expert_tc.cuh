// What the tensor-core kernels of the routed experts share: TMA copies and descriptors of 128-byte-swizzled
// operands, the three-bfloat16 split of 32-bit values, operands in memory and their tensor maps.
#pragma once

#include <cuda.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "num.cuh"
#include "tc_common.cuh"

namespace fsc {
namespace {

constexpr int kSlabRow = 128;  // bytes of a slab row: 64 two-byte elements

// Tile copies into this block's shared memory, where `issue` is not 0 (see elect_one).  PAIR: the block is one of a
// cta_group::2 pair and `bar` (a shared::cluster address) may be its partner's.
template <bool PAIR = false>
__device__ __forceinline__ void tma_tile4(uint32_t issue, uint32_t dst, const CUtensorMap* m, int c0, int c1, int c2, int c3,
                                          uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %7, 0;\n\t"
        "@q cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, "
        "%3, %4, %5}], [%6];\n\t}" ::"r"(dst),
        "l"(m), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar), "r"(issue)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %7, 0;\n\t"
        "@q cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];\n\t}" ::"r"(dst),
        "l"(m), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar), "r"(issue)
        : "memory");
}
template <bool PAIR = false>
__device__ __forceinline__ void tma_tile3(uint32_t issue, uint32_t dst, const CUtensorMap* m, int c0, int c1, int c2,
                                          uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, "
        "%3, %4}], [%5];\n\t}" ::"r"(dst),
        "l"(m), "r"(c0), "r"(c1), "r"(c2), "r"(bar), "r"(issue)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "@q cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];\n\t}" ::"r"(dst),
        "l"(m), "r"(c0), "r"(c1), "r"(c2), "r"(bar), "r"(issue)
        : "memory");
}
__device__ __forceinline__ void expect_if(uint32_t issue, uint64_t* bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%1], %0;\n\t}" ::"r"(bytes),
      "r"(tc::smem_u32(bar)), "r"(issue)
      : "memory");
}

// A pair of blocks (a cluster of two): ranks, addresses in the first block, barriers.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_first_block(uint32_t saddr) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(saddr));
  return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// x as the sum of three bfloat16, exactly: its 24 significand bits cut after 8, 16 and 24 (the planes' bits
// are the upper halves of the words).  Cutting needs no care near the largest float and five instructions;
// with rounded planes the products left out are half as large, which no result shows.
__device__ __forceinline__ void split3(float x, uint32_t* p) {
  const uint32_t h = __float_as_uint(x) & 0xffff0000u;
  const float r = x - __uint_as_float(h);
  const uint32_t m = __float_as_uint(r) & 0xffff0000u;
  p[0] = h, p[1] = m, p[2] = __float_as_uint(r - __uint_as_float(m));
}
// x as the sum of two bfloat16: the first of its upper eight significand bits (cut, or rounded: then the rest is half as
// large, and exact for a value of eleven bits), the second the rest, rounded to 2^-16 of x.  An infinity has no rest.
template <bool CUT>
__device__ __forceinline__ void split2(float x, uint32_t* p) {
  const float h = CUT ? __uint_as_float(__float_as_uint(x) & 0xffff0000u) : __bfloat162float(__float2bfloat16_rn(x));
  const float r = fabsf(h) == INFINITY ? 0.f : x - h;
  p[0] = __float_as_uint(h), p[1] = __float_as_uint(__bfloat162float(__float2bfloat16_rn(r)));
}

// Eight values as 16 bytes of each plane.
__device__ __forceinline__ void split8(const float* v, uint4* q) {
  uint32_t w[3][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t a[3], b[3];
    split3(v[2 * i], a);
    split3(v[2 * i + 1], b);
#pragma unroll
    for (int p = 0; p < 3; ++p) w[p][i] = __byte_perm(a[p], b[p], 0x7632);
  }
#pragma unroll
  for (int p = 0; p < 3; ++p) q[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
}

// Shared-memory matrix descriptor, 128-byte swizzle: `sbo` bytes between groups of eight slab rows;
// MN-major operands wider than 64 elements continue `lbo` bytes on.
__device__ __forceinline__ uint64_t desc128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)((lbo >> 4) & 0x3FFF) << 16 |
         (uint64_t)((sbo >> 4) & 0x3FFF) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// One lane of a converged warp: 1 there, 0 elsewhere.  The warp that issues products runs its loop with all
// lanes and predicates the instructions with this: descriptors then live in uniform registers (moved there
// one by one from a single thread's branch, each product took 123 cycles to issue).
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p;
}

// PAIR: one product of 256 rows of A over the shared memory of both blocks of a pair, issued by the first.
template <typename T, bool PAIR = false>
__device__ __forceinline__ void mma_ss(uint32_t issue, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
#define FSC_MMA(group, kind)                                                                                      \
  asm volatile(                                                                                                  \
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"                              \
      "@q tcgen05.mma." group "." kind " [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),         \
      "r"(accumulate), "r"(issue)                                                                                \
      : "memory")
  if constexpr (PAIR) {
    if constexpr (sizeof(T) == 1) FSC_MMA("cta_group::2", "kind::f8f6f4");
    else FSC_MMA("cta_group::2", "kind::f16");
  } else {
    if constexpr (sizeof(T) == 1) FSC_MMA("cta_group::1", "kind::f8f6f4");
    else FSC_MMA("cta_group::1", "kind::f16");
  }
#undef FSC_MMA
}
// Arrives on `bar` (PAIR: of both blocks) when the products issued so far are done.
template <bool PAIR = false>
__device__ __forceinline__ void commit_if(uint32_t issue, uint64_t* bar) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}" ::"r"(
            tc::smem_u32(bar)),
        "r"(issue), "h"((uint16_t)3)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(tc::smem_u32(bar)),
        "r"(issue)
        : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tmem_take(uint32_t* slot) {  // all 512 columns; one warp
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tc::smem_u32(slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tc::tmem_alloc(slot, 512);
    tc::tmem_relinquish();
  }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_give(uint32_t at) {
  if constexpr (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(at) : "memory");
  else
    tc::tmem_dealloc(at, 512);
}

// Instruction descriptor: fp32 accumulator; f16 = 0 / bf16 = 1 (e4m3 = 0); bits 15 and 16: A and B MN-major.
template <typename T>
__device__ __forceinline__ uint32_t idesc_of(int n, bool a_mn, bool b_mn, int m = 128) {
  constexpr uint32_t fmt = std::is_same<T, __half>::value || sizeof(T) == 1 ? 0 : 1;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// ---- when a bounded wait runs out
// The plan's status word then holds a code, every role gives up, and what the block had still to write is NaN: wrong
// numbers would not show.  A plan whose status is not 0 when a kernel starts gives NaN throughout.  Before the block
// ends, copies and products in flight are waited for, again with a limit.
__device__ __forceinline__ float failed_value() { return __uint_as_float(0x7fc00000u); }

// Alike in the whole warp.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, int32_t* status, int where) {
  return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, status, where));
}

__device__ __noinline__ bool drain(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (clock64() - t0 < tc::kWaitCycles)
    if (tc::mbar_try_wait(bar, parity)) return true;
  return false;
}

// Where there is no barrier of this block to wait on: half a millisecond, hundreds of times what a copy takes.
__device__ __noinline__ void drain_time() {
  const long long t0 = clock64();
  while (clock64() - t0 < 1000000) __nanosleep(1000);
}

// The last expert whose start is at or before `at` (starts ascend; at < start[experts]).
__device__ __forceinline__ int find_expert(const int32_t* start, int experts, int at) {
  int lo = 0, hi = experts;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= at) lo = mid; else hi = mid;
  }
  return lo;
}

// Eight elements of a row of T as 16 bytes of each plane (one, three bfloat16 of 32-bit values, two of 16-bit values that
// may be scaled; 8-bit elements: sixteen as one).  VEC: whole 16-byte pieces, else element by element.
template <typename T, typename E, int P, bool VEC>
struct Piece {
  static constexpr int N = 16 / sizeof(E);
  alignas(16) T v[N];

  __device__ __forceinline__ void load(const T* row, bool live, int c, int cols) {
    if constexpr (VEC) {
      constexpr int L = 16 / sizeof(T);
#pragma unroll
      for (int b = 0; b < N; b += L) {
        uint4 q = make_uint4(0, 0, 0, 0);
        if (live && c + b < cols) q = __ldg(reinterpret_cast<const uint4*>(row + c + b));
        *reinterpret_cast<uint4*>(&v[b]) = q;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        memset(&v[i], 0, sizeof(T));
        if (live && c + i < cols) v[i] = row[c + i];
      }
    }
  }
  __device__ __forceinline__ void store(bool scaled, float f, E* out, int64_t plane) {
    if constexpr (P == 3) {
      if (scaled) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= f;
      }
      uint4 h[3];
      split8(v, h);
#pragma unroll
      for (int q = 0; q < 3; ++q) *reinterpret_cast<uint4*>(out + q * plane) = h[q];
    } else if constexpr (P == 2) {
      uint32_t w[2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a[2], b[2];
        if (scaled) {
          split2<true>(to_f32(v[2 * i]) * f, a);
          split2<true>(to_f32(v[2 * i + 1]) * f, b);
        } else {
          split2<false>(to_f32(v[2 * i]), a);
          split2<false>(to_f32(v[2 * i + 1]), b);
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) w[q][i] = __byte_perm(a[q], b[q], 0x7632);
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) *reinterpret_cast<uint4*>(out + q * plane) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
    } else {
      *reinterpret_cast<uint4*>(out) = *reinterpret_cast<uint4*>(v);  // as it is: 16- and 8-bit rows are not scaled here
    }
  }
};

// Rows as they are, with a pitch that is a multiple of 16 bytes and in planes.
template <typename T, typename E, int P, bool VEC>
__global__ void __launch_bounds__(256) pack_kernel(const T* in, int64_t rows, int cols, int pitch, E* out) {
  constexpr int N = 16 / sizeof(E);
  const int per = pitch / N;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * per; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * N;
    Piece<T, E, P, VEC> p;
    p.load(in + r * cols, true, c, cols);
    p.store(false, 1.f, out + r * pitch + c, rows * pitch);
  }
}

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                            const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

Encode tensor_map_encoder() {
  static const Encode fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<Encode>(p);
  }();
  return fn;
}

template <typename E>
constexpr CUtensorMapDataType map_type() {
  return sizeof(E) == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                        : std::is_same<E, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

// An operand in memory: `planes` of [outer][rows][cols], rows `pitch` elements apart.
template <typename E>
struct Operand {
  const E* p;
  int64_t outer, rows;
  int cols, pitch, planes;
};

template <typename E>
int encode(CUtensorMap* m, const Operand<E>& o, int dims, const cuuint64_t* size, const cuuint64_t* stride,
           const cuuint32_t* box) {
  const Encode fn = tensor_map_encoder();
  if (!fn) return fail(FSC_ERR_CUDA, "expert_linear: cuTensorMapEncodeTiled is not available");
  const cuuint32_t one[4] = {1, 1, 1, 1};
  if (fn(m, map_type<E>(), dims, const_cast<E*>(o.p), size, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return fail(FSC_ERR_CUDA, "expert_linear: cuTensorMapEncodeTiled failed");
  return FSC_OK;
}

// Tiles of `box_rows` rows by 128 bytes: of an expert's weights, or of sorted rows.
template <typename E>
int tile_map(CUtensorMap* m, const Operand<E>& o, int box_rows, bool experts) {
  const cuuint64_t row = (cuuint64_t)o.pitch * sizeof(E);
  if (experts) {
    const cuuint64_t size[4] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)o.outer, (cuuint64_t)o.planes};
    const cuuint64_t stride[3] = {row, row * o.rows, row * o.rows * o.outer};
    const cuuint32_t box[4] = {(cuuint32_t)(kSlabRow / sizeof(E)), (cuuint32_t)box_rows, 1, 1};
    return encode(m, o, 4, size, stride, box);
  }
  const cuuint64_t size[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)o.planes};
  const cuuint64_t stride[2] = {row, row * o.rows};
  const cuuint32_t box[3] = {(cuuint32_t)(kSlabRow / sizeof(E)), (cuuint32_t)box_rows, 1};
  return encode(m, o, 3, size, stride, box);
}

int sm_count() {
  int dev = 0, n = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

// The operand type of T's products, its planes, and elements in 16 bytes.
template <typename T>
struct Of {
  using E = typename std::conditional<sizeof(T) == 4, __nv_bfloat16, T>::type;
  static constexpr int P = sizeof(T) == 4 ? 3 : 1;
  static constexpr int ALIGN = 16 / sizeof(E);
  static int pitch(int64_t cols) { return (int)(ceil_div(cols, ALIGN) * ALIGN); }
  static bool direct(int64_t cols) { return sizeof(T) != 4 && cols % ALIGN == 0; }
};

// Weights as an operand: as they are, or packed into the arena.
template <typename T>
int weights_operand(const T* in, int64_t experts, int64_t rows, int64_t cols, Arena& arena, Operand<typename Of<T>::E>* o,
                    cudaStream_t st) {
  using E = typename Of<T>::E;
  constexpr int P = Of<T>::P;
  *o = Operand<E>{reinterpret_cast<const E*>(in), experts, rows, (int)cols, Of<T>::pitch(cols), P};
  if (Of<T>::direct(cols)) return FSC_OK;
  const int64_t n = experts * rows;
  E* buf = arena.take<E>(P * n * o->pitch);
  o->p = buf;
  if (arena.measuring) return FSC_OK;
  FSC_REQUIRE(arena.ok(), "expert_linear: workspace too small");
  const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(n * (o->pitch / Of<T>::ALIGN), 256), 148 * 8);
  if (cols % (16 / sizeof(T)) == 0)
    pack_kernel<T, E, P, true><<<blocks, 256, 0, st>>>(in, n, (int)cols, o->pitch, buf);
  else
    pack_kernel<T, E, P, false><<<blocks, 256, 0, st>>>(in, n, (int)cols, o->pitch, buf);
  return check_launch("expert_linear pack");
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
  FSC_REQUIRE(z.tokens * z.per_token * z.comps < (1ll << 31) / 3 - 256, "expert_linear: too many rows");
  return FSC_OK;
}


bool al16(std::initializer_list<const void*> ps) {
  uintptr_t all = 0;
  for (const void* p : ps) all |= reinterpret_cast<uintptr_t>(p);
  return (all & 15) == 0;
}

template <typename F>
int by_type(int dtype, F f) {
  if (dtype == FSC_F32) return f(float{});
  if (dtype == FSC_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}

bool float_type(int dtype) { return dtype == FSC_F32 || dtype == FSC_BF16 || dtype == FSC_F16; }

}  // namespace
}  // namespace fsc
