// Experts' products of a few rows (single tokens of a serving step): matrix-vector products.
//
//   out[t, k, :] = sum_j w[t, j] W_e(t, j) x[t, k, :], or the products of each slot apart
//
// Bound by reading the experts' weights once: 8 experts of 2048 x 1024 bf16 are 33.5 MB (5 us of bytes; 11.8 us from a
// cold cache, half of it the chain index, row of W, sum).  A block takes one to four outputs of one token and all of its
// slots (as few as one wave of four blocks per SM allows); each warp streams rows of W, 16 bytes a lane and eight loads
// in flight, the first of them before the token's rows are put into shared memory as fp32, and the slots' sums meet in
// shared memory in the order of the slots.  No plan, no workspace, one launch.
// Tokens that share an expert read it again from the L2, so it is taken for up to 32 slots only.  Measured against the
// plan and the sorted rows, us: 8 of 64 experts of 2048 x 1024 bf16, 8 / 16 / 32 / 64 slots: 10 / 16 / 29 / 54 to
// 23 / 27 / 38 / 49; 2 of 8 experts of 1024 x 1024 bf16, 8 / 16 / 32 / 64 slots: 8 / 13 / 23 / 43 to 17 each; 4 of 16
// experts of 2048 x 2048 fp32, 32 / 64 / 128 slots: 67 / 130 / 254 to 211 each.
#include <type_traits>

#include "common.cuh"
#include "num.cuh"

namespace fsc {
namespace {

constexpr int kMostOutputs = 4, kWarps = 8, kMostComps = 16;
constexpr int kMostX = 12288;  // fp32 values of x in shared memory
constexpr int kMostSlots = 32;

struct FewArgs {
  const void* x;
  const void* w;
  const int32_t* indices;
  const float* weights;  // or null: the slots apart
  const float* x_scale;  // 8 bits
  const float* w_scale;
  void* out;
  int experts, per_token, comps, inputs, outputs;
  int by_slot;
  int per_block;  // outputs of a block
};

template <typename T>
__device__ __forceinline__ float value(T v) {
  return to_f32(v);
}
template <>
__device__ __forceinline__ float value<e4m3>(e4m3 v) {
  uint32_t h;
  const uint16_t two = v.b;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
  return __half2float(__ushort_as_half((uint16_t)h));
}

// Sixteen bytes as fp32.
template <typename T>
__device__ __forceinline__ void values(uint4 q, float* v) {
  if constexpr (sizeof(T) == 1) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t h;
      const uint16_t two = (uint16_t)(w[i / 2] >> (i % 2 * 16));
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
      v[2 * i] = __half2float(__ushort_as_half((uint16_t)h));
      v[2 * i + 1] = __half2float(__ushort_as_half((uint16_t)(h >> 16)));
    }
  } else {
    const T* t = reinterpret_cast<const T*>(&q);
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(T); ++i) v[i] = to_f32(t[i]);
  }
}

// KB: components rounded up (1, 4, 16); VEC: rows of W in 16-byte pieces.
template <typename T, typename OUT, int KB, bool VEC>
__global__ void __launch_bounds__(kWarps * 32) few_kernel(FewArgs a) {
  extern __shared__ float xs[];  // [slots of x][comps][inputs], then [per_token][per_block][comps] products
  constexpr int V = VEC ? 16 / sizeof(T) : 1;
  constexpr int U = sizeof(T) == 1 ? 4 : 8;  // pieces of W in flight
  constexpr int STEP = 32 * V * U;
  using P = typename std::conditional<VEC, uint4, T>::type;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t token = blockIdx.y;
  const int o0 = blockIdx.x * a.per_block;
  const int rows = (a.by_slot ? a.per_token : 1) * a.comps, n = rows * a.inputs;
  float* part = xs + (n + 3) / 4 * 4;
  const T* x = static_cast<const T*>(a.x) + token * n;
  const int32_t* indices = a.indices + token * a.per_token;
  const int tasks = a.per_token * a.per_block;  // task t: slot t / per_block, output t % per_block
  // the row of W of a task, null where there is none
  auto row_of = [&](int t) -> const T* {
    if (t >= tasks) return nullptr;
    const int e = indices[t / a.per_block], o = o0 + t % a.per_block;
    return e >= 0 && e < a.experts && o < a.outputs
               ? static_cast<const T*>(a.w) + ((int64_t)e * a.outputs + o) * a.inputs
               : nullptr;
  };
  P q[U];
  auto load = [&](const T* w, int c0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = c0 + u * 32 * V + lane * V;
      if (w != nullptr && c < a.inputs) {
        if constexpr (VEC) q[u] = __ldcs(reinterpret_cast<const uint4*>(w + c));
        else q[u] = w[c];
      }
    }
  };
  int t = warp;
  const T* w = row_of(t);
  load(w, 0);
  if constexpr (VEC) {
    for (int i = tid * V; i < n; i += kWarps * 32 * V) values<T>(*reinterpret_cast<const uint4*>(x + i), xs + i);
  } else {
    for (int i = tid; i < n; i += kWarps * 32) xs[i] = value<T>(x[i]);
  }
  __syncthreads();
  while (t < tasks) {
    const int j = t / a.per_block, o = o0 + t % a.per_block;
    const float* xr = xs + (a.by_slot ? j : 0) * a.comps * a.inputs;
    float acc[KB];
#pragma unroll
    for (int k = 0; k < KB; ++k) acc[k] = 0.f;
    const T* next = row_of(t + kWarps);
    if (w != nullptr) {
      for (int c0 = 0; c0 < a.inputs; c0 += STEP) {
        if (c0 > 0) load(w, c0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c = c0 + u * 32 * V + lane * V;
          if (c >= a.inputs) break;
          float v[V];
          if constexpr (VEC) values<T>(q[u], v);
          else v[0] = value<T>(q[u]);
#pragma unroll
          for (int k = 0; k < KB; ++k) {
            if (k >= a.comps) break;
            const float* xk = xr + k * a.inputs + c;
#pragma unroll
            for (int i = 0; i < V; i += V < 4 ? 1 : 4) {
              if constexpr (V >= 4) {
                const float4 f = *reinterpret_cast<const float4*>(xk + i);
                acc[k] = fmaf(v[i], f.x, acc[k]);
                acc[k] = fmaf(v[i + 1], f.y, acc[k]);
                acc[k] = fmaf(v[i + 2], f.z, acc[k]);
                acc[k] = fmaf(v[i + 3], f.w, acc[k]);
              } else {
                acc[k] = fmaf(v[i], xk[i], acc[k]);
              }
            }
          }
        }
      }
    }
    load(next, 0);  // on its way while the warp sums
    if (sizeof(T) == 1 && w != nullptr) {
      const int e = indices[j];
      acc[0] *= a.x_scale[a.by_slot ? token * a.per_token + j : token] * a.w_scale[(int64_t)e * a.outputs + o];
    }
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      if (k >= a.comps) break;
      const float d = warp_sum(acc[k]);
      if (lane == 0) part[t * a.comps + k] = d;
    }
    w = next;
    t += kWarps;
  }
  __syncthreads();
  OUT* out = static_cast<OUT*>(a.out);
  const int p = a.per_block;
  if (a.weights) {
    for (int i = tid; i < p * a.comps; i += kWarps * 32) {
      const int k = i / p, o = i % p;
      if (o0 + o >= a.outputs) continue;
      float y = 0.f;
      for (int j = 0; j < a.per_token; ++j) {
        const int e = indices[j];
        if (e >= 0 && e < a.experts) y = fmaf(a.weights[token * a.per_token + j], part[(j * p + o) * a.comps + k], y);
      }
      out[(token * a.comps + k) * a.outputs + o0 + o] = from_f32<OUT>(y);
    }
  } else {
    for (int i = tid; i < a.per_token * p * a.comps; i += kWarps * 32) {
      const int o = i % p, k = i / p % a.comps, j = i / p / a.comps;
      if (o0 + o < a.outputs)
        out[((token * a.per_token + j) * a.comps + k) * a.outputs + o0 + o] = from_f32<OUT>(part[(j * p + o) * a.comps + k]);
    }
  }
}

template <typename T, typename OUT, int KB>
int launch_kb(FewArgs a, int64_t tokens, cudaStream_t st) {
  a.per_block = 1;  // one wave of four blocks per SM where that is enough
  while (a.per_block < kMostOutputs && ceil_div(a.outputs, a.per_block) * tokens > 148 * 4) a.per_block *= 2;
  const int n = (a.by_slot ? a.per_token : 1) * a.comps * a.inputs;
  const size_t smem = ((size_t)(n + 3) / 4 * 4 + (size_t)a.per_token * a.per_block * a.comps) * sizeof(float);
  const dim3 grid((unsigned)ceil_div(a.outputs, a.per_block), (unsigned)tokens);
  const bool vec = a.inputs % (16 / sizeof(T)) == 0 && a.inputs % 4 == 0;
  auto go = [&](auto kernel) {
    constexpr size_t most = (kMostX + kMostSlots * kMostOutputs * kMostComps) * sizeof(float);
    if (smem > 48 * 1024 && !allow_shared(kernel, most)) return check_launch("expert_linear");
    kernel<<<grid, kWarps * 32, smem, st>>>(a);
    return check_launch("expert_linear few rows");
  };
  return vec ? go(few_kernel<T, OUT, KB, true>) : go(few_kernel<T, OUT, KB, false>);
}

template <typename T, typename OUT>
int launch(const FewArgs& a, int64_t tokens, cudaStream_t st) {
  if (a.comps == 1) return launch_kb<T, OUT, 1>(a, tokens, st);
  if constexpr (sizeof(T) == 1) return fail(FSC_ERR_ARGUMENT, "expert_linear_few: 8-bit rows have one component");
  else return a.comps <= 4 ? launch_kb<T, OUT, 4>(a, tokens, st) : launch_kb<T, OUT, kMostComps>(a, tokens, st);
}

}  // namespace
}  // namespace fsc

using namespace fsc;

extern "C" {

int fsc_expert_few_fits(int64_t tokens, int64_t per_token, int64_t comps, int64_t inputs, int x_by_slot) {
  if (tokens < 1 || per_token < 1 || per_token > kMostSlots || comps < 1 || comps > kMostComps || inputs < 1) return 0;
  return tokens <= kMostSlots && tokens * per_token <= kMostSlots && inputs <= kMostX &&
         (x_by_slot ? per_token : 1) * comps * inputs <= kMostX;
}

int fsc_expert_linear_few(int dtype, int out_dtype, const void* x, const float* x_scale, const void* w, const float* w_scale,
                          const int32_t* indices, const float* weights, void* out, int64_t tokens, int64_t per_token,
                          int64_t comps, int64_t experts, int64_t inputs, int64_t outputs, int x_by_slot, void* stream) {
  const bool q8 = dtype == FSC_E4M3;
  FSC_REQUIRE(q8 || dtype == FSC_F32 || dtype == FSC_BF16 || dtype == FSC_F16, "expert_linear_few: dtype");
  FSC_REQUIRE(q8 ? out_dtype == FSC_F32 || out_dtype == FSC_BF16 || out_dtype == FSC_F16 : out_dtype == dtype,
              "expert_linear_few: out_dtype");
  FSC_REQUIRE(experts >= 1 && experts <= 1024 && outputs >= 1 && outputs <= (1 << 20), "expert_linear_few: experts or outputs out of range");
  if (tokens == 0) return FSC_OK;
  FSC_REQUIRE(fsc_expert_few_fits(tokens, per_token, comps, inputs, x_by_slot),
              "expert_linear_few: at most 32 slots, 16 components and 12288 values of x for a token");
  FSC_REQUIRE(!q8 || comps == 1, "expert_linear_few: 8-bit rows have one component");
  FSC_REQUIRE(x && w && indices && out && (!q8 || (x_scale && w_scale)), "expert_linear_few: null pointer");
  FSC_REQUIRE(((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(x)) & 15) == 0,
              "expert_linear_few: x and w must start on 16 bytes");
  FewArgs a{x,      w,   indices,          weights,     x_scale,      w_scale,
            out,    (int)experts, (int)per_token, (int)comps, (int)inputs, (int)outputs,
            x_by_slot != 0, 1};
  cudaStream_t st = as_stream(stream);
  if (q8) {
    if (out_dtype == FSC_F32) return launch<e4m3, float>(a, tokens, st);
    if (out_dtype == FSC_BF16) return launch<e4m3, __nv_bfloat16>(a, tokens, st);
    return launch<e4m3, __half>(a, tokens, st);
  }
  if (dtype == FSC_F32) return launch<float, float>(a, tokens, st);
  if (dtype == FSC_BF16) return launch<__nv_bfloat16, __nv_bfloat16>(a, tokens, st);
  return launch<__half, __half>(a, tokens, st);
}

}  // extern "C"
