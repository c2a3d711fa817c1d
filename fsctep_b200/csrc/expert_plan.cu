// Groups the (token, choice) slots of a routing by expert, and its tokens by the whole choice: stable
// counting sorts.
//
//   offsets[b] .. offsets[b + 1]: the places of bin b in `order`, which lists items in ascending order.
// Slots: bin = expert; slots whose index is outside [0, experts) belong to no bin and are left out.
// Tokens (joint): bin = the choices as digits in base experts + 1, the last digit value for "no expert".
// The order is the same every time (ranks come from ballots over consecutive items, never from the order
// of atomics), so that sums over an expert's rows are too.  Bound by the latency of a chain of dependent
// instructions: a block takes 4096 items, a warp 128 of them, in registers from the load to the place.
// Up to 4096 items it is one launch; beyond, the blocks' counts come first, and every block adds up
// those before it.  Both groupings share the launches.  16,384 slots take 12 us in two
// launches (one block for all took 34 us, a warp's match.any about as long as its ballots).
#include <algorithm>

#include "common.cuh"
#include "num.cuh"

namespace fsc {
namespace {

constexpr int kRounds = 4;  // groups of 32 items that a lane keeps
constexpr int64_t kBlockItems = 1024 * kRounds;
constexpr int64_t kMostBins = 1024;

struct Grouping {
  const int32_t* indices;
  int64_t items;    // 0: nothing to do
  int experts;
  int digits;       // 0: the index itself; else a token's choices
  int bins, bits;   // bits of a bin
  int blocks;
  int32_t* counts;  // [blocks][bins]
  int32_t* offsets;
  int32_t* order;
};

struct PlanArgs {
  Grouping g[2];
  int32_t* status;
};

__device__ __forceinline__ int bin_of(const Grouping& g, int64_t item) {
  if (item >= g.items) return -1;
  if (g.digits == 0) {
    const int e = g.indices[item];
    return e >= 0 && e < g.experts ? e : -1;
  }
  int key = 0;
  for (int j = 0; j < g.digits; ++j) {
    const int e = g.indices[item * g.digits + j];
    key = key * (g.experts + 1) + (e >= 0 && e < g.experts ? e : g.experts);
  }
  return key;
}

// A lane's items of one piece: bin (-1: none), rank among the equal bins of its group of 32 and their number.
// Groups past the last item are skipped, the whole warp alike.
struct Items {
  int bin[kRounds], rank[kRounds];
};

__device__ __forceinline__ void load_items(const Grouping& g, int64_t first, int rounds, Items& it) {
#pragma unroll
  for (int r = 0; r < kRounds; ++r) it.bin[r] = r < rounds ? bin_of(g, first + r * 32 + (threadIdx.x & 31)) : -1;
}

// Lanes with the same bin: one ballot for each bit of the bins (match.any takes several times as long).
__device__ __forceinline__ unsigned same_bin(int bin, int bits) {
  unsigned same = __ballot_sync(0xffffffffu, bin >= 0);
  if (bin < 0) same = 0;
  for (int i = 0; i < bits; ++i) {
    const unsigned m = __ballot_sync(0xffffffffu, bin >> i & 1);
    same &= bin >> i & 1 ? m : ~m;
  }
  return same;
}

// One warp counts its items into `hist` (its own row: no other warp writes it).
__device__ __forceinline__ void count_items(Items& it, int rounds, int bits, int32_t* hist) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if (r >= rounds) break;
    const unsigned same = same_bin(it.bin[r], bits);
    const int rank = __popc(same & ((1u << lane) - 1));
    it.rank[r] = rank | __popc(same) << 8;
    if (it.bin[r] >= 0 && rank == 0) hist[it.bin[r]] += __popc(same);
    __syncwarp();
  }
}

// One warp places its items; next[b]: the next place of bin b for this warp.
__device__ __forceinline__ void place_items(const Grouping& g, int64_t first, const Items& it, int rounds, int32_t* next) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if (r >= rounds) break;
    const int b = it.bin[r], rank = it.rank[r] & 255;
    const int at = b >= 0 ? next[b] : 0;
    __syncwarp();
    if (b >= 0) {
      g.order[at + rank] = (int32_t)(first + r * 32 + lane);
      if (rank == 0) next[b] = at + (it.rank[r] >> 8);
    }
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

__global__ void __launch_bounds__(1024) plan_count_kernel(PlanArgs a) {
  extern __shared__ int32_t hist[];
  const Grouping& g = a.g[blockIdx.y];
  if ((int)blockIdx.x >= g.blocks) return;
  int bin[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) bin[r] = bin_of(g, blockIdx.x * kBlockItems + r * 1024 + threadIdx.x);
  for (int b = threadIdx.x; b < g.bins; b += 1024) hist[b] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
    if (bin[r] >= 0) atomicAdd(&hist[bin[r]], 1);
  __syncthreads();
  for (int b = threadIdx.x; b < g.bins; b += 1024) g.counts[(int64_t)blockIdx.x * g.bins + b] = hist[b];
}

__global__ void __launch_bounds__(1024) plan_place_kernel(PlanArgs a) {
  extern __shared__ int32_t hist[];  // [32][bins], then the items of each bin before this block and in all
  __shared__ int sums[32];
  const Grouping& g = a.g[blockIdx.y];
  if ((int)blockIdx.x >= g.blocks) return;
  const int warp = threadIdx.x >> 5, bins = g.bins, b = threadIdx.x;
  int32_t *before = hist + 32 * bins, *all = before + bins;
  if (b == 0 && blockIdx.x == 0 && blockIdx.y == 0) *a.status = 0;
  const int64_t left = g.items - (int64_t)blockIdx.x * kBlockItems;
  const int rounds = left >= kBlockItems ? kRounds : (int)((left + 1023) / 1024);  // the items spread over all warps
  const int64_t first = (int64_t)blockIdx.x * kBlockItems + (int64_t)warp * rounds * 32;
  Items it;
  load_items(g, first, rounds, it);
  for (int i = b; i < 34 * bins; i += 1024) hist[i] = 0;
  __syncthreads();
  if (g.blocks > 1)
    for (int i = b; i < g.blocks * bins; i += 1024) {
      const int n = g.counts[i];
      if (n) {
        atomicAdd(&all[i % bins], n);
        if (i < (int)blockIdx.x * bins) atomicAdd(&before[i % bins], n);
      }
    }
  count_items(it, rounds, g.bits, hist + warp * bins);
  __syncthreads();
  int sum = 0;
  if (b < bins) {
#pragma unroll 8
    for (int c = 0; c < 32; ++c) {
      const int n = hist[c * bins + b];
      hist[c * bins + b] = sum;
      sum += n;
    }
    if (g.blocks > 1) sum = all[b];
  }
  int total;
  const int start = block_exclusive(sum, sums, &total);
  if (b < bins) {
    if (blockIdx.x == 0) g.offsets[b] = start;
    const int at = start + before[b];
#pragma unroll 8
    for (int c = 0; c < 32; ++c) hist[c * bins + b] += at;
  }
  if (b == 0 && blockIdx.x == 0) g.offsets[bins] = total;
  __syncthreads();
  place_items(g, first, it, rounds, hist + warp * bins);
}

Grouping grouping(int64_t items, int experts, int digits, int bins) {
  Grouping g{};
  g.items = items, g.experts = experts, g.digits = digits, g.bins = bins;
  while ((1 << g.bits) < bins) ++g.bits;
  g.blocks = (int)std::max<int64_t>(1, ceil_div(items, kBlockItems));
  return g;
}

}  // namespace

// Bins of the tokens' whole choices, or 0 where they are too many (over 1024: histograms and the products' tables lie in
// shared memory) or each has too few of the tokens (under 16) to share a tile.  Plan, forward and gradients of narrow
// rows by whole choice and in sorted rows, us: 2 of 8 experts, 9 x 64 fp32, 2 / 8 / 16 / 128 tokens a bin: 30 / 31 / 32 /
// 68 to 32 / 42 / 59 / 295; 2 of 31 experts (1,024 bins), 4 x 64 fp32, 2 / 4 / 8 / 16: 75 / 89 / 92 / 93 to
// 54 / 87 / 143 / 209; 1 of 8 experts, 128 fp32, 16 / 128: 35 / 39 to 29 / 33 (few tokens at all: launches).
int64_t joint_bins(int64_t tokens, int64_t per_token, int64_t experts) {
  int64_t bins = 1;
  for (int64_t j = 0; j < per_token; ++j) {
    bins *= experts + 1;
    if (bins > kMostBins) return 0;
  }
  return tokens >= 16 * bins ? bins : 0;
}

}  // namespace fsc

using namespace fsc;

extern "C" {

int64_t fsc_expert_joint_bins(int64_t tokens, int64_t per_token, int64_t experts) {
  if (tokens < 1 || per_token < 1 || experts < 1) return 0;
  return joint_bins(tokens, per_token, experts);
}

size_t fsc_expert_plan_workspace_bytes(int64_t tokens, int64_t per_token, int64_t experts) {
  if (tokens < 1 || per_token < 1 || experts < 1 || tokens * per_token <= kBlockItems) return 0;
  const int64_t bins = joint_bins(tokens, per_token, experts);
  return (size_t)(ceil_div(tokens * per_token, kBlockItems) * experts + ceil_div(tokens, kBlockItems) * bins) *
         sizeof(int32_t);
}

int fsc_expert_plan(const int32_t* indices, int64_t tokens, int64_t per_token, int64_t experts, int32_t* offsets,
                    int32_t* order, int32_t* joint_offsets, int32_t* joint_order, int32_t* status, void* workspace,
                    size_t workspace_bytes, void* stream) {
  FSC_REQUIRE(experts >= 1 && experts <= 1024, "expert_plan: 1 to 1024 experts");
  FSC_REQUIRE(tokens >= 0 && tokens < (1ll << 31) && per_token >= 1 && per_token <= 32 && tokens * per_token < (1ll << 31),
              "expert_plan: slots out of range");
  const int64_t slots = tokens * per_token;
  FSC_REQUIRE(status && (slots == 0 || indices), "expert_plan: null pointer");
  FSC_REQUIRE((offsets || joint_offsets) && !(offsets && slots && !order) && !(joint_offsets && !joint_order),
              "expert_plan: null pointer");
  FSC_REQUIRE(!joint_offsets || joint_bins(tokens, per_token, experts) > 0, "expert_plan: no joint grouping for these sizes");
  FSC_REQUIRE(workspace_bytes >= fsc_expert_plan_workspace_bytes(tokens, per_token, experts) &&
                  (workspace || slots <= kBlockItems),
              "expert_plan: workspace too small");
  cudaStream_t st = as_stream(stream);
  PlanArgs a{};
  a.status = status;
  int n = 0, most = 0;
  int32_t* counts = static_cast<int32_t*>(workspace);
  auto add = [&](Grouping g, int32_t* off, int32_t* ord) {
    g.indices = indices, g.offsets = off, g.order = ord, g.counts = counts;
    if (counts) counts += (int64_t)g.blocks * g.bins;
    most = std::max(most, g.bins);
    a.g[n++] = g;
  };
  if (offsets) add(grouping(slots, (int)experts, 0, (int)experts), offsets, order);
  if (joint_offsets)
    add(grouping(tokens, (int)experts, (int)per_token, (int)joint_bins(tokens, per_token, experts)), joint_offsets,
        joint_order);
  const dim3 blocks((unsigned)std::max(a.g[0].blocks, a.g[1].blocks), n);
  if (blocks.x > 1) {
    plan_count_kernel<<<blocks, 1024, (size_t)most * sizeof(int32_t), st>>>(a);
    FSC_TRY(check_launch("expert_plan"));
  }
  const size_t smem = 34 * (size_t)most * sizeof(int32_t);
  if (smem > 48 * 1024 && !allow_shared(plan_place_kernel, 34 * kMostBins * sizeof(int32_t)))
    return check_launch("expert_plan");
  plan_place_kernel<<<blocks, 1024, smem, st>>>(a);
  return check_launch("expert_plan");
}

}  // extern "C"
