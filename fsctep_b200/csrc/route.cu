// Routing to experts: scores, an optional balance bias, groups, top-k, renormalised weights; and the
// gradient of the weights in the logits.
//
//   p = softmax(l) or sigmoid(l);  t = p + bias;  a group's score is the sum of its two best t;
//   the top_k best t in the best groups;  w = scale * p_sel [/ (sum p_sel + 1e-20)]
//   gradient: renormalised d_j = scale (g_j - sum_i g_i p_i / S) / S, else d_j = scale g_j;
//   softmax dl = p (d - sum d p), sigmoid dl = d p (1 - p)
//
// One warp owns a token, expert e = 32 i + lane in its registers.  The choice is exact: without bias and
// groups it goes by the logits (p grows with them), else by t in 64 bits, because two scores 1e-8 apart
// decide which expert's weights a token meets.  A score is held as an unsigned key of the same order
// (0: not available), so a warp finds its best with integer maximum reductions, two of 32 bits and one
// for the lowest index among equals.  Bound by memory for large batches (each logit read once), by
// the chain of top_k reductions for one token.
#include <type_traits>

#include "common.cuh"
#include "num.cuh"

namespace fsc {
namespace {

struct RouteArgs {
  const void* logits;
  int64_t stride;
  const float* bias;
  const uint8_t* row_mask;  // 0: the row takes no expert; null: every row does
  float* weights;
  int32_t* indices;
  const float* grad_weights;  // backward
  void* grad_logits;
  int64_t tokens;
  int experts, top_k, groups, kept;
  int softmax, renormalize;
  float scale;
};

constexpr unsigned kAll = 0xffffffffu;

// Unsigned keys in the order of the values; every value but NaN maps above 0.
__device__ __forceinline__ uint32_t key32(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t key64(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double value64(uint64_t k) {
  return __longlong_as_double((long long)(k >> 63 ? k ^ 0x8000000000000000ull : ~k));
}

__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(kAll, k); }
__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(kAll, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(kAll, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return (uint64_t)hi << 32 | lo;
}

// A logit as the operator takes it: -inf and NaN are not available, +inf is the largest float.
template <typename T>
__device__ __forceinline__ bool logit_of(const T* row, int e, float& l) {
  l = to_f32(row[e]);
  const bool ok = l > -INFINITY;
  l = ok ? fminf(l, 3.402823466e38f) : -INFINITY;
  return ok;
}

// Softmax statistics of a row: the maximum and the sum of exp(l - max).
template <int NX, typename S>
__device__ __forceinline__ void softmax_stats(const float* l, float& top, S& sum) {
  top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NX; ++i) top = fmaxf(top, l[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
  sum = 0;
  if (top == -INFINITY) return;
#pragma unroll
  for (int i = 0; i < NX; ++i) sum += exp((S)l[i] - (S)top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
}

template <typename T, int NX, typename K>
__global__ void __launch_bounds__(128) route_kernel(RouteArgs a) {
  constexpr bool WIDE = sizeof(K) == 8;  // choice by 64-bit scores (bias or groups), else by the logits
  using S = typename std::conditional<WIDE, double, float>::type;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= a.tokens) return;
  float* wout = a.weights + row * a.top_k;
  int32_t* iout = a.indices + row * a.top_k;
  if (a.row_mask && a.row_mask[row] == 0) {
    if (lane < a.top_k) wout[lane] = 0.f, iout[lane] = -1;
    return;
  }
  const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
  float l[NX];
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    const int e = i * 32 + lane;
    l[i] = -INFINITY;
    if (e < a.experts) logit_of(logits, e, l[i]);
  }
  float top = 0.f;
  S sum = 1;
  if (a.softmax) softmax_stats<NX, S>(l, top, sum);
  K key[NX];
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    const int e = i * 32 + lane;
    key[i] = 0;
    if (l[i] > -INFINITY) {
      if constexpr (WIDE) {
        double t = a.softmax ? exp((double)l[i] - (double)top) / sum : 1.0 / (1.0 + exp(-(double)l[i]));
        if (a.bias) t += (double)a.bias[e];
        key[i] = t > -INFINITY ? key64(t) : 0;  // a bias of -inf or NaN closes an expert
      } else {
        key[i] = key32(l[i]);
      }
    }
  }
  if constexpr (WIDE) {
    if (a.groups > 1 && a.kept < a.groups) {
      // lane g holds group g's score (groups <= 32)
      const int per = a.experts / a.groups;
      uint64_t mine = 0;
      for (int g = 0; g < a.groups; ++g) {
        const int lo = g * per, hi = lo + per;
        K b1 = 0, b2 = 0;  // the lane's two best in the group
#pragma unroll
        for (int i = 0; i < NX; ++i) {
          const int e = i * 32 + lane;
          if (e >= lo && e < hi) {
            if (key[i] > b1) b2 = b1, b1 = key[i];
            else if (key[i] > b2) b2 = key[i];
          }
        }
        const K m1 = warp_max(b1);
        const unsigned who = __ballot_sync(kAll, b1 == m1);
        const K m2 = warp_max(lane == __ffs(who) - 1 ? b2 : b1);
        if (lane == g && m1) {
          const double s = m2 ? value64(m1) + value64(m2) : value64(m1);
          mine = s == s ? key64(s) : key64(-INFINITY);  // inf - inf: behind every other group
        }
      }
      unsigned open = 0;  // bit g: group g is kept
      for (int j = 0; j < a.kept; ++j) {
        const uint64_t m = warp_max(mine);
        if (m == 0) break;
        const int g = __ffs(__ballot_sync(kAll, mine == m)) - 1;
        open |= 1u << g;
        if (lane == g) mine = 0;
      }
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const int e = i * 32 + lane;
        if (e < a.experts && !(open >> (e / per) & 1)) key[i] = 0;
      }
    }
  }
  // top_k: each lane offers its best; the winner's lane looks for its next one
  K best = 0;
  int at = 0;
  auto refresh = [&] {
    best = 0, at = 0;
#pragma unroll
    for (int i = 0; i < NX; ++i)
      if (key[i] > best) best = key[i], at = i;  // the first of equals: the lowest index of the lane
  };
  refresh();
  int pick = -1;
  for (int j = 0; j < a.top_k; ++j) {
    const K m = warp_max(best);
    if (m == 0) break;
    const int e = (int)__reduce_min_sync(kAll, best == m ? (unsigned)(at * 32 + lane) : 0xffffffffu);
    if (lane == j) pick = e;
    if (lane == (e & 31)) {
#pragma unroll
      for (int i = 0; i < NX; ++i)
        if (i == (e >> 5)) key[i] = 0;
      refresh();
    }
  }
  // the chosen scores without the bias, one per lane
  S p = 0;
  if (pick >= 0) {
    float v;
    logit_of(logits, pick, v);
    p = a.softmax ? exp((S)v - (S)top) / sum : (S)1 / ((S)1 + exp(-(S)v));
  }
  if (a.renormalize) {
    S total = p;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(kAll, total, o);
    p /= total + (S)1e-20;
  }
  if (lane < a.top_k) {
    wout[lane] = pick >= 0 ? (float)(p * (S)a.scale) : 0.f;
    iout[lane] = pick;
  }
}

template <typename T, int NX>
__global__ void __launch_bounds__(128) route_backward_kernel(RouteArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= a.tokens) return;
  const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
  T* out = static_cast<T*>(a.grad_logits) + row * a.experts;
  int pick = lane < a.top_k ? a.indices[row * a.top_k + lane] : -1;
  if (pick >= a.experts) pick = -1;
  const bool any = __any_sync(kAll, pick >= 0);
  float l[NX], d[NX];
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    const int e = i * 32 + lane;
    l[i] = -INFINITY, d[i] = 0.f;
    if (any && e < a.experts) logit_of(logits, e, l[i]);
  }
  float top = 0.f, sum = 1.f;
  if (any && a.softmax) softmax_stats<NX, float>(l, top, sum);
  float p = 0.f, g = 0.f;
  if (pick >= 0) {
    float v;
    if (!logit_of(logits, pick, v)) pick = -1;
    else p = a.softmax ? expf(v - top) / sum : 1.f / (1.f + expf(-v));
    g = a.grad_weights[row * a.top_k + lane] * a.scale;
    if (pick < 0) g = 0.f;
  }
  if (a.renormalize) {
    const float total = warp_sum(p) + 1e-20f, gp = warp_sum(g * p);
    g = pick >= 0 ? (g - gp / total) / total : 0.f;
  }
  const float dot = a.softmax ? warp_sum(g * p) : 0.f;
  for (int j = 0; j < a.top_k; ++j) {
    const int e = __shfl_sync(kAll, pick, j);
    const float ge = __shfl_sync(kAll, g, j);
    if (e >= 0 && (e & 31) == lane) {
#pragma unroll
      for (int i = 0; i < NX; ++i)
        if (i == (e >> 5)) d[i] += ge;
    }
  }
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    const int e = i * 32 + lane;
    if (e >= a.experts) continue;
    float v = 0.f;
    if (any && l[i] > -INFINITY) {
      const float q = a.softmax ? expf(l[i] - top) / sum : 1.f / (1.f + expf(-l[i]));
      v = a.softmax ? q * (d[i] - dot) : d[i] * q * (1.f - q);
    }
    out[e] = from_f32<T>(v);
  }
}

template <typename T, int NX>
int launch_nx(const RouteArgs& a, bool back, bool wide, cudaStream_t st) {
  const unsigned blocks = (unsigned)ceil_div(a.tokens, 4);
  if (back)
    route_backward_kernel<T, NX><<<blocks, 128, 0, st>>>(a);
  else if (wide)
    route_kernel<T, NX, uint64_t><<<blocks, 128, 0, st>>>(a);
  else
    route_kernel<T, NX, uint32_t><<<blocks, 128, 0, st>>>(a);
  return check_launch("route_experts");
}

template <typename T>
int launch_t(const RouteArgs& a, bool back, bool wide, cudaStream_t st) {
  const int nx = (int)ceil_div(a.experts, 32);
  if (nx <= 1) return launch_nx<T, 1>(a, back, wide, st);
  if (nx <= 2) return launch_nx<T, 2>(a, back, wide, st);
  if (nx <= 4) return launch_nx<T, 4>(a, back, wide, st);
  if (nx <= 8) return launch_nx<T, 8>(a, back, wide, st);
  if (nx <= 16) return launch_nx<T, 16>(a, back, wide, st);
  return launch_nx<T, 32>(a, back, wide, st);
}

int launch(int dtype, const RouteArgs& a, bool back, bool wide, cudaStream_t st) {
  if (dtype == FSC_F32) return launch_t<float>(a, back, wide, st);
  if (dtype == FSC_BF16) return launch_t<__nv_bfloat16>(a, back, wide, st);
  return launch_t<__half>(a, back, wide, st);
}

int check(int dtype, int64_t tokens, int64_t experts, int64_t top_k, int scores) {
  FSC_REQUIRE(dtype == FSC_F32 || dtype == FSC_BF16 || dtype == FSC_F16, "route_experts: dtype must be f32, bf16 or f16");
  FSC_REQUIRE(tokens >= 0 && tokens < (1ll << 31), "route_experts: tokens out of range");
  FSC_REQUIRE(experts >= 1 && experts <= 1024, "route_experts: 1 to 1024 experts");
  FSC_REQUIRE(top_k >= 1 && top_k <= 32 && top_k <= experts, "route_experts: top_k must be 1 to 32 and at most the experts");
  FSC_REQUIRE(scores == 0 || scores == 1, "route_experts: scores must be 0 (softmax) or 1 (sigmoid)");
  return FSC_OK;
}

}  // namespace
}  // namespace fsc

using namespace fsc;

extern "C" {

int fsc_route_experts(int dtype, const void* logits, int64_t stride, const float* bias, const uint8_t* row_mask,
                      float* weights, int32_t* indices, int64_t tokens, int64_t experts, int64_t top_k, int64_t groups,
                      int64_t groups_kept, int scores, int renormalize, float scale, void* stream) {
  FSC_TRY(check(dtype, tokens, experts, top_k, scores));
  FSC_REQUIRE(groups >= 1 && groups <= 32 && experts % groups == 0, "route_experts: 1 to 32 groups that divide the experts");
  FSC_REQUIRE(groups_kept >= 1 && groups_kept <= groups, "route_experts: groups_kept must be 1 to the groups");
  FSC_REQUIRE(top_k <= experts / groups * groups_kept, "route_experts: top_k exceeds the kept groups' experts");
  if (tokens == 0) return FSC_OK;
  FSC_REQUIRE(logits && weights && indices, "route_experts: null pointer");
  RouteArgs a{};
  a.logits = logits, a.stride = stride, a.bias = bias, a.row_mask = row_mask, a.weights = weights, a.indices = indices;
  a.tokens = tokens, a.experts = (int)experts, a.top_k = (int)top_k, a.groups = (int)groups, a.kept = (int)groups_kept;
  a.softmax = scores == 0, a.renormalize = renormalize != 0, a.scale = scale;
  return launch(dtype, a, false, bias != nullptr || groups_kept < groups, as_stream(stream));
}

int fsc_route_experts_backward(int dtype, const float* grad_weights, const void* logits, int64_t stride,
                               const int32_t* indices, void* grad_logits, int64_t tokens, int64_t experts,
                               int64_t top_k, int scores, int renormalize, float scale, void* stream) {
  FSC_TRY(check(dtype, tokens, experts, top_k, scores));
  if (tokens == 0) return FSC_OK;
  FSC_REQUIRE(grad_weights && logits && indices && grad_logits, "route_experts_backward: null pointer");
  RouteArgs a{};
  a.logits = logits, a.stride = stride, a.indices = const_cast<int32_t*>(indices), a.grad_weights = grad_weights;
  a.grad_logits = grad_logits, a.tokens = tokens, a.experts = (int)experts, a.top_k = (int)top_k;
  a.softmax = scores == 0, a.renormalize = renormalize != 0, a.scale = scale;
  return launch(dtype, a, true, false, as_stream(stream));
}

}  // extern "C"
