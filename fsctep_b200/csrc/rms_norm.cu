// Root-mean-square norm of a row with the residual's addition, its 8-bit form and its gradient.
//
//   s = x + r,  u = 1 / sqrt(mean(s^2) + eps),  y = s u g,  h = s rounded to the rows' type
//   8 bits: c = max|y| / 448, q = e4m3(y / c)
//   gradient, from the stored h: a = dy g,  n = h u,  dx = u (a - n mean(a n)) + dh,  dg = sum_rows dy n
//   (u mean(a h) in place of mean(a n); u^3 would leave the range of fp32 for rows of 1e13 or, without eps, 1e-13)
//
// Bound by memory: every tensor is read or written once.  A row stays in the registers of the threads
// that own it (a warp for short rows, so that no barrier is needed and many rows are in flight per
// SM; a block for long ones) between the reduction and the output; rows too long for that are read
// a second time.  The sum s is normalised before it is rounded, all sums are 32-bit, and each
// output is rounded once.  16384 x 4096 bf16 rows with a residual take 90 us (6.0 TB/s, 91 % of a measured copy),
// 8191 x 2048 with 8-bit output 26 us, the gradient of 64000 x 576 fp32 rows 95 us and 4 us for the weight's.
#include <algorithm>

#include "common.cuh"
#include "num.cuh"

namespace fsc {
namespace {

struct NormArgs {
  const void* x;         // forward: x; backward: h
  const void* r;         // forward: residual or null; backward: grad_h or null
  const void* gy;        // backward: grad_y
  const void* w;
  int64_t x_stride, r_stride, gy_stride;
  void* y;               // forward: y; backward: grad_x
  void* h;               // forward: x + residual, or null
  uint8_t* q;            // 8-bit form: quantised rows (then y is null)
  float* scale;
  float* partial;        // backward: [gridDim.x][dim] column sums, or null
  float eps;
  int64_t rows;
  int dim;
};

// Sum (or maximum) over the threads that own a row: a warp, or the whole block.
template <int TPR, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* smem) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? (t > v || t != t ? t : v) : v + t;  // a NaN wins the maximum, so that it reaches the scale
  }
  if constexpr (TPR > 32) {
    constexpr int NW = TPR / 32;
    const int lane = threadIdx.x & 31;
    __syncthreads();  // smem may still be read by the previous reduction
    if (lane == 0) smem[threadIdx.x >> 5] = v;
    __syncthreads();
    v = smem[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) {
      const float t = smem[i];
      v = MAX ? (t > v || t != t ? t : v) : v + t;
    }
  }
  return v;
}

// Outputs are written once and not read here: they leave the caches first.
template <typename V>
__device__ __forceinline__ void store_stream(void* p, const V& v) {
  if constexpr (sizeof(V) == 16)
    __stcs(static_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&v));
  else
    *static_cast<V*>(p) = v;
}

template <int VE, typename W>
__device__ __forceinline__ void load_weight(const void* w, int c, float* out) {
  constexpr int N = sizeof(W) * VE > 16 ? 16 / sizeof(W) : VE;
#pragma unroll
  for (int b = 0; b < VE; b += N) {
    const Pack<W, N> p = *reinterpret_cast<const Pack<W, N>*>(static_cast<const W*>(w) + c + b);
#pragma unroll
    for (int i = 0; i < N; ++i) out[b + i] = to_f32(p.v[i]);
  }
}

template <int VE>
__device__ __forceinline__ void store_e4m3(uint8_t* dst, const float* v) {
  if constexpr (VE == 1) {
    *dst = static_cast<uint8_t>(e4m3x2(v[0], 0.f) & 0xFF);
  } else {
    Pack<uint16_t, VE / 2> p;
#pragma unroll
    for (int i = 0; i < VE / 2; ++i) p.v[i] = e4m3x2(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<Pack<uint16_t, VE / 2>*>(dst) = p;
  }
}

// The row lives in registers: TPR threads, NV vectors of VE elements each.
template <typename T, typename W, int VE, int TPR, int NV>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR) norm_forward_kernel(NormArgs a) {
  __shared__ float smem[32];
  const int t = TPR == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t row = TPR == 32 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  if (row >= a.rows) return;  // whole warps, and never in a block that synchronises
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* r = a.r ? static_cast<const T*>(a.r) + row * a.r_stride : nullptr;
  using V = Pack<T, VE>;
  V xv[NV], rv[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * VE;
    if (c < a.dim) {
      xv[i] = *reinterpret_cast<const V*>(x + c);
      if (r) rv[i] = *reinterpret_cast<const V*>(r + c);
    }
  }
  float s[NV][VE];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * VE;
    if (c < a.dim) {
      V hv;
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        s[i][j] = to_f32(xv[i].v[j]) + (r ? to_f32(rv[i].v[j]) : 0.f);
        ss = fmaf(s[i][j], s[i][j], ss);
        hv.v[j] = from_f32<T>(s[i][j]);
      }
      if (a.h) store_stream(static_cast<T*>(a.h) + row * a.dim + c, hv);
    } else {
#pragma unroll
      for (int j = 0; j < VE; ++j) s[i][j] = 0.f;
    }
  }
  ss = row_reduce<TPR, false>(ss, smem);
  const float u = __frsqrt_rn(ss / (float)a.dim + a.eps);
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * VE;
    if (c < a.dim) {
      float g[VE];
      load_weight<VE, W>(a.w, c, g);
      V yv;
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float y = s[i][j] * u * g[j];
        s[i][j] = y;
        yv.v[j] = from_f32<T>(y);
        const float m = fabsf(y);
        top = m > top || m != m ? m : top;
      }
      if (a.y) store_stream(static_cast<T*>(a.y) + row * a.dim + c, yv);
    }
  }
  if (!a.q) return;
  top = row_reduce<TPR, true>(top, smem);
  const float scale = top / 448.f;
  if (t == 0) a.scale[row] = scale;
  // times the reciprocal, which is off by a unit of 32 bits where e4m3 keeps four; a scale whose reciprocal could
  // overflow divides
  const float inv = scale > 1e-30f ? __frcp_rn(scale) : 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * VE;
    if (c < a.dim) {
      if (inv > 0.f) {
#pragma unroll
        for (int j = 0; j < VE; ++j) s[i][j] *= inv;
      } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) s[i][j] = scale == 0.f ? 0.f : s[i][j] / scale;
      }
      store_e4m3<VE>(a.q + row * a.dim + c, s[i]);
    }
  }
}

// Rows too long for the registers of a block: the row is read once for each pass over it.
template <typename T, typename W>
__global__ void __launch_bounds__(1024) norm_forward_long_kernel(NormArgs a) {
  __shared__ float smem[32];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* r = a.r ? static_cast<const T*>(a.r) + row * a.r_stride : nullptr;
  const W* w = static_cast<const W*>(a.w);
  auto at = [&](int c) { return to_f32(x[c]) + (r ? to_f32(r[c]) : 0.f); };
  float ss = 0.f;
  for (int c = threadIdx.x; c < a.dim; c += 1024) {
    const float s = at(c);
    ss = fmaf(s, s, ss);
    if (a.h) static_cast<T*>(a.h)[row * a.dim + c] = from_f32<T>(s);
  }
  ss = row_reduce<1024, false>(ss, smem);
  const float u = __frsqrt_rn(ss / (float)a.dim + a.eps);
  float top = 0.f;
  for (int c = threadIdx.x; c < a.dim; c += 1024) {
    const float y = at(c) * u * to_f32(w[c]);
    const float m = fabsf(y);
    top = m > top || m != m ? m : top;
    if (a.y) static_cast<T*>(a.y)[row * a.dim + c] = from_f32<T>(y);
  }
  if (!a.q) return;
  top = row_reduce<1024, true>(top, smem);
  const float scale = top / 448.f;
  if (threadIdx.x == 0) a.scale[row] = scale;
  for (int c = threadIdx.x; c < a.dim; c += 1024) {
    const float y = at(c) * u * to_f32(w[c]);
    const float v = scale == 0.f ? 0.f : y / scale;
    store_e4m3<1>(a.q + row * a.dim + c, &v);
  }
}

// Gradient.  Every thread keeps the same columns for all rows that it meets, so the weight's
// gradient is summed in registers; each block writes one partial row, and a second kernel adds them
// in block order (no atomics: the result does not depend on timing).
template <typename T, typename W, int VE, int TPR, int NV>
__global__ void __launch_bounds__(TPR == 32 ? 128 : TPR) norm_backward_kernel(NormArgs a) {
  constexpr int RPB = TPR == 32 ? 4 : 1;  // rows of a block at a time
  extern __shared__ float dyn[];          // RPB > 1: [4][dim] partial sums
  __shared__ float smem[32];
  const int t = TPR == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const int sub = TPR == 32 ? (threadIdx.x >> 5) : 0;
  using V = Pack<T, VE>;
  float acc[NV][VE];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j) acc[i][j] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * RPB + sub; row < a.rows; row += (int64_t)gridDim.x * RPB) {
    const T* h = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* gy = static_cast<const T*>(a.gy) + row * a.gy_stride;
    const T* gh = a.r ? static_cast<const T*>(a.r) + row * a.r_stride : nullptr;
    V hv[NV], yv[NV], rv[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VE;
      if (c < a.dim) {
        hv[i] = *reinterpret_cast<const V*>(h + c);
        yv[i] = *reinterpret_cast<const V*>(gy + c);
        if (gh) rv[i] = *reinterpret_cast<const V*>(gh + c);
      }
    }
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VE;
      if (c < a.dim) {
        float g[VE];
        load_weight<VE, W>(a.w, c, g);
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float hf = to_f32(hv[i].v[j]);
          ss = fmaf(hf, hf, ss);
          dot = fmaf(to_f32(yv[i].v[j]) * g[j], hf, dot);
        }
      }
    }
    ss = row_reduce<TPR, false>(ss, smem);
    dot = row_reduce<TPR, false>(dot, smem);
    const float u = __frsqrt_rn(ss / (float)a.dim + a.eps);
    const float k = u * dot / (float)a.dim;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VE;
      if (c < a.dim) {
        float g[VE];
        load_weight<VE, W>(a.w, c, g);
        V out;
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float hf = to_f32(hv[i].v[j]), yf = to_f32(yv[i].v[j]);
          const float n = hf * u;
          float d = u * fmaf(-n, k, yf * g[j]);
          if (gh) d += to_f32(rv[i].v[j]);
          out.v[j] = from_f32<T>(d);
          acc[i][j] = fmaf(yf, n, acc[i][j]);
        }
        if (a.y) store_stream(static_cast<T*>(a.y) + row * a.dim + c, out);
      }
    }
  }
  if (!a.partial) return;
  float* dst = RPB > 1 ? dyn + (int64_t)sub * a.dim : a.partial + (int64_t)blockIdx.x * a.dim;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * VE;
    if (c < a.dim)
#pragma unroll
      for (int j = 0; j < VE; ++j) dst[c + j] = acc[i][j];
  }
  if constexpr (RPB > 1) {
    __syncthreads();
    for (int c = threadIdx.x; c < a.dim; c += 128)
      a.partial[(int64_t)blockIdx.x * a.dim + c] = (dyn[c] + dyn[a.dim + c]) + (dyn[2 * a.dim + c] + dyn[3 * a.dim + c]);
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(1024) norm_backward_long_kernel(NormArgs a) {
  __shared__ float smem[32];
  const W* w = static_cast<const W*>(a.w);
  float* part = a.partial ? a.partial + (int64_t)blockIdx.x * a.dim : nullptr;
  if (part)
    for (int c = threadIdx.x; c < a.dim; c += 1024) part[c] = 0.f;  // each column has one owner thread
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* h = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* gy = static_cast<const T*>(a.gy) + row * a.gy_stride;
    const T* gh = a.r ? static_cast<const T*>(a.r) + row * a.r_stride : nullptr;
    float ss = 0.f, dot = 0.f;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
      const float hf = to_f32(h[c]);
      ss = fmaf(hf, hf, ss);
      dot = fmaf(to_f32(gy[c]) * to_f32(w[c]), hf, dot);
    }
    ss = row_reduce<1024, false>(ss, smem);
    dot = row_reduce<1024, false>(dot, smem);
    const float u = __frsqrt_rn(ss / (float)a.dim + a.eps);
    const float k = u * dot / (float)a.dim;
    for (int c = threadIdx.x; c < a.dim; c += 1024) {
      const float hf = to_f32(h[c]), yf = to_f32(gy[c]);
      const float n = hf * u;
      float d = u * fmaf(-n, k, yf * to_f32(w[c]));
      if (gh) d += to_f32(gh[c]);
      if (a.y) static_cast<T*>(a.y)[row * a.dim + c] = from_f32<T>(d);
      if (part) part[c] = fmaf(yf, n, part[c]);
    }
  }
}

// dg[c] = sum over the blocks' partial rows, in order; 32 threads share a column.
template <typename W>
__global__ void __launch_bounds__(1024) norm_weight_sum_kernel(const float* partial, int parts, int dim, W* out) {
  __shared__ float sm[32][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
  float s = 0.f;
  if (c < dim)
    for (int p = g; p < parts; p += 32) s += partial[(int64_t)p * dim + c];
  sm[g][threadIdx.x & 31] = s;
  __syncthreads();
  s = warp_sum(sm[threadIdx.x & 31][g]);  // warp g: column g of the block
  const int mine = blockIdx.x * 32 + g;
  if ((threadIdx.x & 31) == 0 && mine < dim) out[mine] = from_f32<W>(s);
}

constexpr int kWarpVectors = 5;

int backward_blocks(int64_t rows, bool warp_rows) {
  // 148 SMs: four blocks of four rows each, or four blocks of one long row, resident per SM
  return (int)std::min<int64_t>(warp_rows ? ceil_div(rows, 4) : rows, 148 * 4);
}

template <typename T, typename W, int VE, bool BACK, int TPR, int NV>
int launch_one(const NormArgs& a, cudaStream_t st) {
  if (BACK) {
    const int blocks = backward_blocks(a.rows, TPR == 32);
    const size_t dyn = TPR == 32 && a.partial ? (size_t)a.dim * 16 : 0;
    norm_backward_kernel<T, W, VE, TPR, NV><<<blocks, TPR == 32 ? 128 : TPR, dyn, st>>>(a);
  } else {
    const int64_t blocks = TPR == 32 ? ceil_div(a.rows, 4) : a.rows;
    norm_forward_kernel<T, W, VE, TPR, NV><<<(unsigned)blocks, TPR == 32 ? 128 : TPR, 0, st>>>(a);
  }
  return check_launch("rms_norm");
}

template <typename T, typename W, int VE, bool BACK>
int launch_ve(const NormArgs& a, cudaStream_t st) {
  const int nv = (int)ceil_div(a.dim, VE);
  // A warp per row up to 5 vectors a lane, blocks of 128, 256 and 1024 threads beyond.  Limits of 2 / 5 / 8 vectors, us:
  // 65536 x 640 bf16 (3 a lane) forward 91 / 65 / 66, gradient 150 / 99 / 98; 16384 x 1280 bf16 (5) forward 33 / 31 / 43,
  // gradient 65 / 76 / 95; 16384 x 1536 bf16 (6) 36 / 36 / 47 and 67 / 67 / 112; 64000 x 576 fp32 (5) 89 / 90 / 91 and
  // 139 / 76 / 121.
  if (nv <= 32 * kWarpVectors) {
    switch (ceil_div(nv, 32)) {
      case 1: return launch_one<T, W, VE, BACK, 32, 1>(a, st);
      case 2: return launch_one<T, W, VE, BACK, 32, 2>(a, st);
      case 3: return launch_one<T, W, VE, BACK, 32, 3>(a, st);
      case 4: return launch_one<T, W, VE, BACK, 32, 4>(a, st);
      default: return launch_one<T, W, VE, BACK, 32, kWarpVectors>(a, st);
    }
  }
  if (nv <= 128 * 2) return launch_one<T, W, VE, BACK, 128, 2>(a, st);
  if (nv <= 256 * 2) return launch_one<T, W, VE, BACK, 256, 2>(a, st);
  if (nv <= 256 * 4) return launch_one<T, W, VE, BACK, 256, 4>(a, st);
  if constexpr (!BACK) {
    if (nv <= 1024 * 2) return launch_one<T, W, VE, BACK, 1024, 2>(a, st);
  }
  if (BACK)
    norm_backward_long_kernel<T, W><<<backward_blocks(a.rows, false), 1024, 0, st>>>(a);
  else
    norm_forward_long_kernel<T, W><<<(unsigned)a.rows, 1024, 0, st>>>(a);
  return check_launch("rms_norm");
}

bool warp_rows(int64_t dim, int ve) { return ceil_div(dim, ve) <= 32 * kWarpVectors; }

bool aligned(const void* p, int64_t stride_bytes) {
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)stride_bytes) & 15) == 0;
}

template <typename T, typename W, bool BACK>
int launch_typed(const NormArgs& a, bool vec, cudaStream_t st) {
  constexpr int VE = 16 / sizeof(T);
  return vec ? launch_ve<T, W, VE, BACK>(a, st) : launch_ve<T, W, 1, BACK>(a, st);
}

template <bool BACK>
int launch(int dtype, int wdtype, const NormArgs& a, bool vec, cudaStream_t st) {
  if (dtype == FSC_F32) return launch_typed<float, float, BACK>(a, vec, st);
  if (dtype == FSC_BF16)
    return wdtype == FSC_F32 ? launch_typed<__nv_bfloat16, float, BACK>(a, vec, st)
                             : launch_typed<__nv_bfloat16, __nv_bfloat16, BACK>(a, vec, st);
  return wdtype == FSC_F32 ? launch_typed<__half, float, BACK>(a, vec, st)
                           : launch_typed<__half, __half, BACK>(a, vec, st);
}

int check_types(int dtype, int wdtype, int64_t rows, int64_t dim) {
  FSC_REQUIRE(dtype == FSC_F32 || dtype == FSC_BF16 || dtype == FSC_F16, "rms_norm: dtype must be f32, bf16 or f16");
  FSC_REQUIRE(wdtype == dtype || wdtype == FSC_F32, "rms_norm: the weight has the rows' dtype or f32");
  FSC_REQUIRE(rows >= 0 && rows < (1ll << 31), "rms_norm: rows out of range");
  FSC_REQUIRE(dim >= 1 && dim <= (1 << 24), "rms_norm: dim must be between 1 and 2^24");
  return FSC_OK;
}

}  // namespace
}  // namespace fsc

using namespace fsc;

extern "C" {

int fsc_rms_norm_forward(int dtype, int weight_dtype, const void* x, int64_t x_stride, const void* residual,
                         int64_t residual_stride, const void* weight, float eps, void* y, void* h, void* q,
                         float* scale, int64_t rows, int64_t dim, void* stream) {
  FSC_TRY(check_types(dtype, weight_dtype, rows, dim));
  if (rows == 0) return FSC_OK;
  FSC_REQUIRE((y != nullptr) != (q != nullptr), "rms_norm: give y or q, not both");
  FSC_REQUIRE((q != nullptr) == (scale != nullptr), "rms_norm: q and scale go together");
  FSC_REQUIRE(x && weight, "rms_norm: null pointer");
  const int64_t es = dtype == FSC_F32 ? 4 : 2;
  NormArgs a{};
  a.x = x, a.r = residual, a.w = weight, a.y = y, a.h = h, a.q = static_cast<uint8_t*>(q), a.scale = scale;
  a.x_stride = x_stride, a.r_stride = residual_stride, a.eps = eps, a.rows = rows, a.dim = (int)dim;
  const bool vec = dim % (16 / es) == 0 && aligned(x, x_stride * es) && aligned(residual, residual_stride * es) &&
                   aligned(weight, 0) && aligned(y, 0) && aligned(h, 0) &&
                   (reinterpret_cast<uintptr_t>(q) & 7) == 0;
  return launch<false>(dtype, weight_dtype, a, vec, as_stream(stream));
}

size_t fsc_rms_norm_backward_workspace_bytes(int64_t rows, int64_t dim) {
  if (rows < 1 || dim < 1) return 0;
  return (size_t)std::min<int64_t>(rows, 148 * 4) * (size_t)dim * sizeof(float);
}

int fsc_rms_norm_backward(int dtype, int weight_dtype, const void* grad_y, int64_t grad_y_stride, const void* grad_h,
                          int64_t grad_h_stride, const void* h, int64_t h_stride, const void* weight, float eps,
                          void* grad_x, void* grad_weight, int64_t rows, int64_t dim, void* workspace,
                          size_t workspace_bytes, void* stream) {
  FSC_TRY(check_types(dtype, weight_dtype, rows, dim));
  cudaStream_t st = as_stream(stream);
  const int64_t es = dtype == FSC_F32 ? 4 : 2, ws = weight_dtype == FSC_F32 ? 4 : 2;
  if (rows == 0) {
    if (grad_weight && cudaMemsetAsync(grad_weight, 0, dim * ws, st) != cudaSuccess) return check_launch("rms_norm");
    return FSC_OK;
  }
  FSC_REQUIRE(grad_y && h && weight, "rms_norm: null pointer");
  FSC_REQUIRE(!grad_weight || (workspace && workspace_bytes >= fsc_rms_norm_backward_workspace_bytes(rows, dim)),
              "rms_norm: workspace too small");
  NormArgs a{};
  a.x = h, a.r = grad_h, a.gy = grad_y, a.w = weight, a.y = grad_x;
  a.partial = grad_weight ? static_cast<float*>(workspace) : nullptr;
  a.x_stride = h_stride, a.r_stride = grad_h_stride, a.gy_stride = grad_y_stride;
  a.eps = eps, a.rows = rows, a.dim = (int)dim;
  const int ve = 16 / es;
  const bool vec = dim % ve == 0 && aligned(h, h_stride * es) && aligned(grad_h, grad_h_stride * es) &&
                   aligned(grad_y, grad_y_stride * es) && aligned(weight, 0) && aligned(grad_x, 0);
  FSC_TRY(launch<true>(dtype, weight_dtype, a, vec, st));
  if (!grad_weight) return FSC_OK;
  const int parts = backward_blocks(rows, warp_rows(dim, vec ? ve : 1));
  const unsigned blocks = (unsigned)ceil_div(dim, 32);
  if (weight_dtype == FSC_F32)
    norm_weight_sum_kernel<float><<<blocks, 1024, 0, st>>>(a.partial, parts, a.dim, static_cast<float*>(grad_weight));
  else if (weight_dtype == FSC_BF16)
    norm_weight_sum_kernel<__nv_bfloat16><<<blocks, 1024, 0, st>>>(a.partial, parts, a.dim,
                                                                  static_cast<__nv_bfloat16*>(grad_weight));
  else
    norm_weight_sum_kernel<__half><<<blocks, 1024, 0, st>>>(a.partial, parts, a.dim, static_cast<__half*>(grad_weight));
  return check_launch("rms_norm weight gradient");
}

}  // extern "C"
