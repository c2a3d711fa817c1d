// Groups the (token, choice) slots of a routing by expert: a stable counting sort.
//
//   offsets[e] .. offsets[e + 1]: the places of expert e in `order`, which lists slots in ascending order.
// Slots whose index is outside [0, experts) belong to no expert and are left out.  The order is the
// same every time (ranks come from warp matches over consecutive slots, never from atomics), so that
// sums over an expert's rows are too.  One block does it all for up to 16,384 slots; beyond that
// three launches: counts of each chunk, their prefix sums, the places.
#include <algorithm>

#include "common.cuh"

namespace fsc {
namespace {

constexpr int kChunksOne = 32;      // chunks (warps) of the one-block form
constexpr int64_t kOneBlock = 16384;
constexpr int kMostChunks = 1024;

struct PlanArgs {
  const int32_t* indices;
  int64_t slots;
  int experts;
  int chunk;       // slots of a chunk, a multiple of 32
  int chunks;
  int32_t* counts; // [chunks][experts]
  int32_t* offsets;
  int32_t* order;
  int32_t* status;
};

__device__ __forceinline__ int expert_of(const PlanArgs& a, int64_t slot, int64_t end) {
  if (slot >= end) return -1;
  const int e = a.indices[slot];
  return e >= 0 && e < a.experts ? e : -1;
}

// One warp counts its chunk into `hist` (its own row: no other warp writes it).
__device__ __forceinline__ void count_chunk(const PlanArgs& a, int64_t lo, int64_t hi, int32_t* hist) {
  const int lane = threadIdx.x & 31;
  for (int64_t s = lo; s < hi; s += 32) {
    const int e = expert_of(a, s + lane, hi);
    const unsigned same = __match_any_sync(0xffffffffu, e);
    if (e >= 0 && lane == __ffs(same) - 1) hist[e] += __popc(same);
    __syncwarp();
  }
}

// One warp places its chunk's slots; `next[e]`: the next place of expert e for this chunk.
__device__ __forceinline__ void place_chunk(const PlanArgs& a, int64_t lo, int64_t hi, int32_t* next) {
  const int lane = threadIdx.x & 31;
  for (int64_t s = lo; s < hi; s += 32) {
    const int e = expert_of(a, s + lane, hi);
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1));
    if (e >= 0) a.order[next[e] + rank] = (int32_t)(s + lane);
    __syncwarp();
    if (e >= 0 && rank == 0) next[e] += __popc(same);
    __syncwarp();
  }
}

// Exclusive sum over the block's 1024 threads.
__device__ __forceinline__ int block_exclusive(int v, int* sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += t;
  }
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += t;
    }
    sums[lane] = s;
  }
  __syncthreads();
  *total = sums[31];
  return x - v + (warp ? sums[warp - 1] : 0);
}

__global__ void __launch_bounds__(1024) plan_one_kernel(PlanArgs a) {
  extern __shared__ int32_t hist[];  // [32][experts]
  __shared__ int sums[32];
  const int warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kChunksOne * a.experts; i += 1024) hist[i] = 0;
  if (threadIdx.x == 0) *a.status = 0;
  __syncthreads();
  const int64_t lo = (int64_t)warp * a.chunk, hi = min(lo + a.chunk, a.slots);
  count_chunk(a, lo, hi, hist + warp * a.experts);
  __syncthreads();
  const int e = threadIdx.x;
  int sum = 0;
  if (e < a.experts)
    for (int c = 0; c < kChunksOne; ++c) {
      const int n = hist[c * a.experts + e];
      hist[c * a.experts + e] = sum;
      sum += n;
    }
  int total;
  const int start = block_exclusive(sum, sums, &total);
  if (e < a.experts) {
    a.offsets[e] = start;
    for (int c = 0; c < kChunksOne; ++c) hist[c * a.experts + e] += start;
  }
  if (e == 0) a.offsets[a.experts] = total;
  __syncthreads();
  place_chunk(a, lo, hi, hist + warp * a.experts);
}

__global__ void __launch_bounds__(128) plan_count_kernel(PlanArgs a) {
  const int c = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (c >= a.chunks) return;
  int32_t* hist = a.counts + (int64_t)c * a.experts;
  for (int e = threadIdx.x & 31; e < a.experts; e += 32) hist[e] = 0;
  __syncwarp();
  const int64_t lo = (int64_t)c * a.chunk;
  count_chunk(a, lo, min(lo + a.chunk, a.slots), hist);
}

// counts -> each chunk's first place of each expert (a warp per expert, 32 chunks at a time).
__global__ void __launch_bounds__(1024) plan_scan_kernel(PlanArgs a) {
  __shared__ int sums[32];
  __shared__ int32_t each[1024];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) *a.status = 0;
  for (int e = warp; e < a.experts; e += 32) {
    int base = 0;
    for (int c0 = 0; c0 < a.chunks; c0 += 32) {
      const int c = c0 + lane;
      const int v = c < a.chunks ? a.counts[(int64_t)c * a.experts + e] : 0;
      int x = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += t;
      }
      if (c < a.chunks) a.counts[(int64_t)c * a.experts + e] = base + x - v;
      base += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) each[e] = base;
  }
  __syncthreads();
  int total;
  const int e = threadIdx.x;
  const int start = block_exclusive(e < a.experts ? each[e] : 0, sums, &total);
  if (e < a.experts) a.offsets[e] = start;
  if (e == 0) a.offsets[a.experts] = total;
}

__global__ void __launch_bounds__(128) plan_place_kernel(PlanArgs a) {
  const int c = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (c >= a.chunks) return;
  int32_t* next = a.counts + (int64_t)c * a.experts;
  for (int e = threadIdx.x & 31; e < a.experts; e += 32) next[e] += a.offsets[e];
  __syncwarp();
  const int64_t lo = (int64_t)c * a.chunk;
  place_chunk(a, lo, min(lo + a.chunk, a.slots), next);
}

int chunk_of(int64_t slots) {
  const int64_t least = slots <= kOneBlock ? ceil_div(slots, kChunksOne) : std::max<int64_t>(512, ceil_div(slots, kMostChunks));
  return (int)(ceil_div(std::max<int64_t>(least, 1), 32) * 32);
}

}  // namespace
}  // namespace fsc

using namespace fsc;

extern "C" {

size_t fsc_expert_plan_workspace_bytes(int64_t slots, int64_t experts) {
  if (slots <= kOneBlock || experts < 1) return 0;
  return (size_t)ceil_div(slots, chunk_of(slots)) * (size_t)experts * sizeof(int32_t);
}

int fsc_expert_plan(const int32_t* indices, int64_t slots, int64_t experts, int32_t* offsets, int32_t* order,
                    int32_t* status, void* workspace, size_t workspace_bytes, void* stream) {
  FSC_REQUIRE(experts >= 1 && experts <= 1024, "expert_plan: 1 to 1024 experts");
  FSC_REQUIRE(slots >= 0 && slots < (1ll << 31), "expert_plan: slots out of range");
  FSC_REQUIRE(offsets && status && (slots == 0 || (indices && order)), "expert_plan: null pointer");
  FSC_REQUIRE(workspace_bytes >= fsc_expert_plan_workspace_bytes(slots, experts) && (workspace || slots <= kOneBlock),
              "expert_plan: workspace too small");
  cudaStream_t st = as_stream(stream);
  PlanArgs a{};
  a.indices = indices, a.slots = slots, a.experts = (int)experts, a.chunk = chunk_of(slots);
  a.offsets = offsets, a.order = order, a.status = status, a.counts = static_cast<int32_t*>(workspace);
  if (slots <= kOneBlock) {
    const size_t smem = (size_t)kChunksOne * experts * sizeof(int32_t);
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(plan_one_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
      return check_launch("expert_plan");
    plan_one_kernel<<<1, 1024, smem, st>>>(a);
    return check_launch("expert_plan");
  }
  a.chunks = (int)ceil_div(slots, a.chunk);
  const unsigned blocks = (unsigned)ceil_div(a.chunks, 4);
  plan_count_kernel<<<blocks, 128, 0, st>>>(a);
  plan_scan_kernel<<<1, 1024, 0, st>>>(a);
  plan_place_kernel<<<blocks, 128, 0, st>>>(a);
  return check_launch("expert_plan");
}

}  // extern "C"
