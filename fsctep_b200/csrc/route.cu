// Routing to experts: scores, an optional balance bias, groups, top-k, renormalised weights; and the
// gradient of the weights in the logits.
//
//   p = softmax(l) or sigmoid(l);  t = p + bias;  a group's score is the sum of its two best t;
//   the top_k best t in the best groups;  w = scale * p_sel [/ (sum p_sel + 1e-20)]
//   gradient: renormalised d_j = scale (g_j - sum_i g_i p_i / S) / S, else d_j = scale g_j;
//   softmax dl = p (d - sum d p), sigmoid dl = d p (1 - p)
//
// One warp owns a token, expert e = 32 i + lane in its registers.  The choice is exact: without bias and
// groups it goes by the logits (p grows with them); else by t in 32 bits wherever the scores that decide are
// further apart than their error, and again in 64 bits where they are not (about one token in 600 of 256
// experts; two scores 1e-8 apart decide which expert's weights a token meets).  A score is held as an unsigned
// key of the same order (0: not available), so a warp finds its best with an integer maximum reduction and
// one for the lowest index among equals; with up to eight keys a lane each lane sorts its own and offers
// its first.  Bound by instruction issue for large batches (about 2,000 a token of 256 experts: 1 us per
// round of the top-k, 10 us for the groups, 7 us for the scores of 16,384 tokens), by one token's
// chain for small ones: 16384 x 256 logits with bias and groups take 37 us, 68 us with every score in 64 bits.
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
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k >> 31 ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ double value_of(uint64_t k) {
  return __longlong_as_double((long long)(k >> 63 ? k ^ 0x8000000000000000ull : ~k));
}

__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(kAll, k); }
__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(kAll, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(kAll, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return (uint64_t)hi << 32 | lo;
}

// A logit as the operator takes it: -inf and NaN are not available, +inf is the largest float, and -0 is 0 (adding 0
// makes it so): their scores are equal, which the keys' order would not say.
template <typename T>
__device__ __forceinline__ bool logit_of(const T* row, int e, float& l) {
  l = to_f32(row[e]);
  const bool ok = l > -INFINITY;
  l = ok ? fminf(l, 3.402823466e38f) + 0.f : -INFINITY;
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

// The best score of a warp's keys and its expert, taken out of them; false if none is available.
template <int NX, typename K>
__device__ __forceinline__ bool take_best(K* key, K& m, int& e) {
  const int lane = threadIdx.x & 31;
  K best = 0;
#pragma unroll
  for (int i = 0; i < NX; ++i) best = max(best, key[i]);
  m = warp_max(best);
  int at = 0xffff;
#pragma unroll
  for (int i = NX - 1; i >= 0; --i) at = key[i] == m ? i * 32 : at;  // the first of equals: the lane's lowest index
  e = (int)__reduce_min_sync(kAll, (unsigned)(at + lane));
  const int mine = e - lane;
#pragma unroll
  for (int i = 0; i < NX; ++i) key[i] = i * 32 == mine ? K(0) : key[i];
  return m != 0;
}

// Closes all but the kept best groups by the sum of their two best keys' values; false where two sums that decide are
// closer than `error` (64-bit keys: never).  Lane g reads group g's keys from shared memory (`buf`, the warp's own),
// each lane starting elsewhere in its group so that groups of 32 do not meet in one bank.
template <int NX, typename K, typename S>
__device__ __forceinline__ bool keep_groups(const RouteArgs& a, K* key, K* buf, S error) {
  const int lane = threadIdx.x & 31, per = a.experts / a.groups;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < NX; ++i) buf[i * 32 + lane] = key[i];
  __syncwarp();
  K mine = 0;  // lane g: group g's sum
  if (lane < a.groups) {
    K b1 = 0, b2 = 0;
    auto take = [&](K k) { b2 = max(b2, min(b1, k)), b1 = max(b1, k); };
    const K* k0 = buf + lane * per;
    if (sizeof(K) == 4 && per % 4 == 0) {
      int at = lane * 4 % per;
      for (int i = 0; i < per; i += 4) {
        const uint4 k = *reinterpret_cast<const uint4*>(k0 + at);
        take((K)k.x), take((K)k.y), take((K)k.z), take((K)k.w);
        at = at + 4 == per ? 0 : at + 4;
      }
    } else {
      int at = lane % per;
      for (int i = 0; i < per; ++i) {
        take(k0[at]);
        at = at + 1 == per ? 0 : at + 1;
      }
    }
    if (b1) {
      const S s = b2 ? value_of(b1) + value_of(b2) : value_of(b1);
      mine = s == s ? key_of(s) : key_of((S)-INFINITY);  // inf - inf: behind every other group
    }
  }
  unsigned open = 0;  // bit g: group g is kept
  K last = 0;
  bool sure = true;
  for (int j = 0; j <= a.kept; ++j) {
    const K m = warp_max(mine);
    if (j == a.kept) {  // the best group that is not kept
      if (sizeof(K) == 4 && m) sure = value_of(last) - value_of(m) > error;
      break;
    }
    if (m == 0) break;
    last = m;
    const int g = __ffs(__ballot_sync(kAll, mine == m)) - 1;
    open |= 1u << g;
    if (lane == g) mine = 0;
  }
  const float inv = 1.f / (float)per;  // (e + 1/2) / per, at least 1 / 2048 away from a whole number
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    const int g = (int)((float)(i * 32 + lane) * inv + 0.5f * inv);
    key[i] = open >> (g & 31) & 1 ? key[i] : K(0);  // past the last expert keys are 0 anyway
  }
  return sure;
}

// A lane's keys in descending order (NX a power of two): Batcher's odd-even merge sort.
template <int NX>
__device__ __forceinline__ void sort_keys(uint32_t* k) {
#pragma unroll
  for (int p = 1; p < NX; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int j = q % p; j + q < NX; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < NX && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t a = k[i + j], b = k[i + j + q];
            k[i + j] = max(a, b), k[i + j + q] = min(a, b);
          }
}

// The choice by scores in 64 bits: lane j's expert.
template <typename T, int NX>
__device__ __noinline__ int route_wide(const RouteArgs& a, const T* logits, uint64_t* buf) {
  const int lane = threadIdx.x & 31;
  uint64_t key[NX];
  float l[NX], top = 0.f;
  double sum = 1;
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    const int e = i * 32 + lane;
    l[i] = -INFINITY;
    if (e < a.experts) logit_of(logits, e, l[i]);
  }
  if (a.softmax) softmax_stats<NX, double>(l, top, sum);
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    key[i] = 0;
    if (l[i] > -INFINITY) {
      double t = a.softmax ? exp((double)l[i] - (double)top) / sum : 1.0 / (1.0 + exp(-(double)l[i]));
      if (a.bias) t += (double)a.bias[i * 32 + lane];
      key[i] = t > -INFINITY ? key_of(t) : 0;  // a bias of -inf or NaN closes an expert
    }
  }
  if (a.kept < a.groups) keep_groups<NX, uint64_t, double>(a, key, buf, 0.0);
  int pick = -1;
  for (int j = 0; j < a.top_k; ++j) {
    uint64_t m;
    int e;
    if (!take_best<NX>(key, m, e)) break;
    if (lane == j) pick = e;
  }
  return pick;
}

// WIDE: bias or closed groups, the choice goes by the scores; else by the logits.
template <typename T, int NX, bool WIDE>
__global__ void __launch_bounds__(128, NX <= 8 ? 10 : 4) route_kernel(const __grid_constant__ RouteArgs a) {
  constexpr bool PACKED = WIDE && NX <= 8;
  __shared__ alignas(16) uint64_t buffer[WIDE ? 4 * NX * 32 : 1];
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= a.tokens) return;
  uint64_t* buf = buffer + (WIDE ? (threadIdx.x >> 5) * NX * 32 : 0);
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
  float top = 0.f, sum = 1.f;
  if (a.softmax) softmax_stats<NX, float>(l, top, sum);
  uint32_t key[NX];
  float far = 0.f;  // the largest magnitude of a score
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    key[i] = 0;
    if (l[i] > -INFINITY) {
      if constexpr (WIDE) {
        float t = a.softmax ? __fdividef(__expf(l[i] - top), sum) : __fdividef(1.f, 1.f + __expf(-l[i]));
        if (a.bias) t += a.bias[i * 32 + lane];
        key[i] = t > -INFINITY ? key_of(t) : 0;
        if constexpr (PACKED) key[i] = key[i] ? (key[i] & ~7u) | i : 0;  // a finite score's key stays above 0
        far = t > -INFINITY ? fmaxf(far, fabsf(t)) : far;
      } else {
        key[i] = key_of(l[i]);
      }
    }
  }
  // How far two scores in 32 bits may be off, of the larger magnitude (or 1): an exponential by 2 + 1.2 |l| units, which
  // count times p (1 - p) or p, and a quotient by 2 units, 4e-7; the softmax's sum by half a unit for each of the NX + 4
  // additions, as where terms below half a unit are lost to a sum near 1, 7e-7 for 8 scores a lane and 2.2e-6 for 32
  // (p times that, and two p add up to 1 at most); the sum with the bias by half a unit.  Up to eight scores a lane carry
  // their place i in their three lowest bits, which puts two of them off by up to seven units each, 1.7e-6.
  constexpr float kApart = 3e-6f;
  bool sure = true;
  if constexpr (WIDE) {
    if (a.kept < a.groups) {
      const float most = __uint_as_float(__reduce_max_sync(kAll, __float_as_uint(far)));
      sure = keep_groups<NX, uint32_t, float>(a, key, reinterpret_cast<uint32_t*>(buf), 4.f * kApart * fmaxf(1.f, most));
      sure = sure && most < 1e30f;
    }
  }
  int pick = -1;
  float before = INFINITY;
  if constexpr (PACKED) sort_keys<NX>(key);
  for (int j = 0; j < a.top_k + (WIDE ? 1 : 0); ++j) {
    uint32_t m;
    int e;
    if constexpr (PACKED) {  // every lane offers its first; equal ones are settled in 64 bits
      m = warp_max(key[0]);
      if (m == 0) break;
      const unsigned who = __ballot_sync(kAll, key[0] == m);
      const int lead = __ffs(who) - 1;
      e = (int)(m & 7u) * 32 + lead;
      sure = sure && (who & (who - 1)) == 0;
      const bool mine = lane == lead;
#pragma unroll
      for (int i = 0; i + 1 < NX; ++i) key[i] = mine ? key[i + 1] : key[i];
      key[NX - 1] = mine ? 0 : key[NX - 1];
    } else {
      if (!take_best<NX>(key, m, e)) break;
    }
    if constexpr (WIDE) {
      const float t = value_of(m);
      sure = sure && !(before - t <= kApart * fmaxf(1.f, fabsf(t)));
      sure = sure && (j == 0 || before < 1e30f);
      before = t;
    }
    if (lane == j && j < a.top_k) pick = e;
  }
  if (WIDE && !sure) pick = route_wide<T, NX>(a, logits, buf);
  // the chosen scores without the bias, one per lane
  float p = 0.f;
  if (pick >= 0) {
    float v;
    logit_of(logits, pick, v);
    p = a.softmax ? expf(v - top) / sum : 1.f / (1.f + expf(-v));
  }
  if (a.renormalize) p /= warp_sum(p) + 1e-20f;
  if (lane < a.top_k) {
    wout[lane] = pick >= 0 ? p * a.scale : 0.f;
    iout[lane] = pick;
  }
}

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// In 64 bits up to the result, which is rounded to 32 bits and from there to the logits' type: the renormalised gradient is a difference g_j - mean(g) of often
// nearly equal terms (for top_k 1 of equal ones), and p (1 - p) of a saturated sigmoid one of p and 1.
template <typename T, int NX>
__global__ void __launch_bounds__(128) route_backward_kernel(const __grid_constant__ RouteArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= a.tokens) return;
  const T* logits = static_cast<const T*>(a.logits) + row * a.stride;
  T* out = static_cast<T*>(a.grad_logits) + row * a.experts;
  int pick = lane < a.top_k ? a.indices[row * a.top_k + lane] : -1;
  if (pick >= a.experts) pick = -1;
  const bool any = __any_sync(kAll, pick >= 0);
  float l[NX];
  double d[NX];
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    const int e = i * 32 + lane;
    l[i] = -INFINITY, d[i] = 0.0;
    if (any && e < a.experts) logit_of(logits, e, l[i]);
  }
  float top = 0.f;
  double sum = 1.0;
  if (any && a.softmax) softmax_stats<NX, double>(l, top, sum);
  double p = 0.0, g = 0.0;
  if (pick >= 0) {
    float v;
    if (!logit_of(logits, pick, v)) pick = -1;
    else p = a.softmax ? exp((double)v - (double)top) / sum : 1.0 / (1.0 + exp(-(double)v));
    g = pick < 0 ? 0.0 : (double)a.grad_weights[row * a.top_k + lane] * (double)a.scale;
  }
  if (a.renormalize) {
    const double total = warp_sum64(p) + 1e-20, gp = warp_sum64(g * p);
    g = pick >= 0 ? (g - gp / total) / total : 0.0;
  }
  const double dot = a.softmax ? warp_sum64(g * p) : 0.0;
  for (int j = 0; j < a.top_k; ++j) {
    const int e = __shfl_sync(kAll, pick, j);
    const double ge = __shfl_sync(kAll, g, j);
    if (e >= 0 && (e & 31) == lane) {
#pragma unroll
      for (int i = 0; i < NX; ++i)
        if (i * 32 + lane == e) d[i] += ge;
    }
  }
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    const int e = i * 32 + lane;
    if (e >= a.experts) continue;
    double v = 0.0;
    if (any && l[i] > -INFINITY) {
      if (a.softmax) {
        v = exp((double)l[i] - (double)top) / sum * (d[i] - dot);
      } else if (d[i] != 0.0) {
        const double q = 1.0 / (1.0 + exp(-(double)l[i]));
        v = d[i] * q * (1.0 - q);
      }
    }
    out[e] = from_f32<T>((float)v);
  }
}

template <typename T, int NX>
int launch_nx(const RouteArgs& a, bool back, bool wide, cudaStream_t st) {
  const unsigned blocks = (unsigned)ceil_div(a.tokens, 4);
  if (back)
    route_backward_kernel<T, NX><<<blocks, 128, 0, st>>>(a);
  else if (wide)
    route_kernel<T, NX, true><<<blocks, 128, 0, st>>>(a);
  else
    route_kernel<T, NX, false><<<blocks, 128, 0, st>>>(a);
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
