// Experts' products of narrow rows (up to 128 channels), all choices of a token at once.
//
//   out[t, k, :] = sum_j w[t, j] W_j x[t, k, :],  W_j the matrix of the token's j-th choice
//   gradient:  gx[t, k, :] = sum_j w[t, j] W_j^T g[t, k, :],  gw[t, j] = sum_k <W_j^T g[t, k, :], x[t, k, :]>
//
// Bound by memory: at 64 channels a row is 256 bytes and its products 16 kFLOP.  Taken slot by slot a row
// would be read top_k times and its products written and read again; here tokens are grouped by their
// whole choice (the plan's joint grouping), so a tile of 128 rows meets the same few matrices, is read
// once and written once: 50,021 atoms of 9 x 64 fp32 values through 2 of 8 experts take what their
// bytes take.  A block owns consecutive tiles and keeps the choice's matrices in shared memory until the
// choice changes.  Eight warps load the rows, split them into bfloat16 planes (fp32) and store the
// 128-byte-swizzled operand; one thread issues tcgen05.mma (rows = TMEM lanes) for each choice into columns
// of its own; eight warps join the columns with the token's weights, a row a thread, while the next
// tile's products run.  The five small products of the fp32 form have an accumulator of their own.
#include "expert_joint.cuh"
#include "expert_tc.cuh"

namespace fsc {
namespace {

constexpr int kMostChoices = 4;
constexpr int kMostStages = 3;
constexpr int kSmem = 204800;
constexpr int kJointThreads = 576;  // warps 0-7 rows, 8-15 epilogue, 16 weights, 17 products

struct JointArgs {
  const void* in;        // rows to multiply: x, or the output's gradient
  const void* x;         // gradient: the rows that the products are multiplied with, or null
  const float* weights;  // [tokens][per_token]
  const int32_t* offsets;
  const int32_t* order;
  int32_t* status;
  void* out;
  float* dots;  // gradient: [tokens][per_token], or null
  int bins, experts, per_token, comps;
  int features, Kd;
  int per_tile;  // tokens of a tile
  int stages, buffers;
  int wide;  // rows of out and x in pieces of 16 values, out on 32 bytes
};

struct JointShared {
  uint64_t x_full[kMostStages], x_empty[kMostStages], acc_full[2], acc_empty[2], w_full, w_empty;
  uint32_t tmem;
  int32_t tiles[1025], first[1025];  // tiles and places before each choice
  float dots[2][2][128][kMostChoices];  // [tile parity][column half][row][choice]
};

__device__ __forceinline__ void store8(float* p, const float* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// Sixteen values of a row as T; `whole`: all sixteen exist and the address is a multiple of 32 (fp32) or 16 bytes.
template <typename T>
__device__ __forceinline__ void store16(T* p, const float* v, int n, bool whole) {
  if (whole) {
    if constexpr (sizeof(T) == 4) {
      store8(p, v);
      store8(p + 8, v + 8);
    } else {
#pragma unroll
      for (int b = 0; b < 16; b += 8) {
        Pack<T, 8> q;
#pragma unroll
        for (int i = 0; i < 8; ++i) q.v[i] = from_f32<T>(v[b + i]);
        *reinterpret_cast<Pack<T, 8>*>(p + b) = q;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < n) p[i] = from_f32<T>(v[i]);
  }
}
template <typename T>
__device__ __forceinline__ void load16(const T* p, float* v, int n, bool whole) {
  if (whole) {
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int b = 0; b < 16; b += E) {
      Pack<T, E> q = *reinterpret_cast<const Pack<T, E>*>(p + b);
#pragma unroll
      for (int i = 0; i < E; ++i) v[b + i] = to_f32(q.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = i < n ? to_f32(p[i]) : 0.f;
  }
}

struct JointTile {
  int key, place, count;  // the choice, first place in the order, tokens
};

// Walks the tiles lo .. hi - 1 of a block.
struct Walk {
  int tile, hi, key;
  __device__ Walk(const JointArgs& a, const JointShared& s) {
    const int total = s.tiles[a.bins], per = (total + gridDim.x - 1) / gridDim.x;
    tile = min((int)blockIdx.x * per, total);
    hi = min(tile + per, total);
    key = tile < hi ? find_expert(s.tiles, a.bins, tile) : 0;
  }
  __device__ bool next(const JointArgs& a, const JointShared& s, JointTile& t) {
    if (tile >= hi) return false;
    while (tile >= s.tiles[key + 1]) ++key;
    t.key = key;
    t.place = s.first[key] + (tile - s.tiles[key]) * a.per_tile;
    t.count = min(a.per_tile, s.first[key + 1] - t.place);
    ++tile;
    return true;
  }
};

// The j-th choice of a key (digits in base experts + 1, the first choice the highest), -1: no expert.
__device__ __forceinline__ int choice(const JointArgs& a, int key, int j) {
  for (int i = a.per_token - 1; i > j; --i) key /= a.experts + 1;
  const int e = key % (a.experts + 1);
  return e < a.experts ? e : -1;
}

// T: rows' type, E: operand element, P: planes, NB: features rounded up (64, 128), KS: slabs of 64 contraction
// elements, BACK: W^T and the products with x, VEC: rows in 16-byte pieces.
template <typename T, typename E, int P, int NB, int KS, bool BACK, bool VEC>
__global__ void __launch_bounds__(kJointThreads, 1) joint_kernel(const __grid_constant__ CUtensorMap mw, JointArgs a) {
  constexpr int X_STAGE = P * KS * 128 * kSlabRow, W_PLANE = KS * NB * kSlabRow;
  constexpr int COLS = NB * (P == 3 ? 2 : 1);  // TMEM columns of a choice
  extern __shared__ uint8_t dyn[];
  __shared__ JointShared s;
  const uint32_t base = (tc::smem_u32(dyn) + 1023) & ~1023u, wbase = base + a.stages * X_STAGE;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < kMostStages; ++i) tc::mbar_init(&s.x_full[i], 8), tc::mbar_init(&s.x_empty[i], 1);
    for (int i = 0; i < 2; ++i) tc::mbar_init(&s.acc_full[i], 1), tc::mbar_init(&s.acc_empty[i], 8);
    tc::mbar_init(&s.w_full, 1), tc::mbar_init(&s.w_empty, 1);
    tc::fence_mbar_init();
  }
  for (int b = tid; b <= a.bins; b += kJointThreads) {
    const int here = a.offsets[b];
    s.first[b] = here;
    if (b < a.bins) s.tiles[b + 1] = (a.offsets[b + 1] - here + a.per_tile - 1) / a.per_tile;
  }
  if (warp == 17) {
    tc::tmem_alloc(&s.tmem, 512);
    tc::tmem_relinquish();
  }
  __syncthreads();
  if (warp == 0) {
    int sum = 0;
    for (int b0 = 0; b0 < a.bins; b0 += 32) {
      int x = b0 + lane < a.bins ? s.tiles[b0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += v;
      }
      if (b0 + lane < a.bins) s.tiles[b0 + lane + 1] = sum + x;
      sum += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) s.tiles[0] = 0;
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  Walk walk(a, s);
  JointTile t;
  bool ok = true;
  if (warp < 8) {  // ---- rows
    constexpr int PIECES = 4 * KS, ROW_PIECES = 8 * KS;
    const int c = tid % ROW_PIECES, col = c * 8;
    int where[PIECES];  // token of the tile and component of each piece's row
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int row = tid / ROW_PIECES + i * (256 / ROW_PIECES);
      where[i] = row / a.comps << 16 | row % a.comps;
    }
    T v[PIECES][8];
    int token[PIECES];
    auto tokens = [&](const JointTile& q) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) token[i] = (where[i] >> 16) < q.count ? a.order[q.place + (where[i] >> 16)] : -1;
    };
    auto load = [&] {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const T* row = static_cast<const T*>(a.in) + ((int64_t)token[i] * a.comps + (where[i] & 0xffff)) * a.Kd;
        if constexpr (VEC) {
          constexpr int L = 16 / sizeof(T);
#pragma unroll
          for (int b = 0; b < 8; b += L) {
            uint4 u = make_uint4(0, 0, 0, 0);
            if (token[i] >= 0 && col + b < a.Kd) u = __ldg(reinterpret_cast<const uint4*>(row + col + b));
            *reinterpret_cast<uint4*>(&v[i][b]) = u;
          }
        } else {
#pragma unroll
          for (int b = 0; b < 8; ++b) v[i][b] = token[i] >= 0 && col + b < a.Kd ? row[col + b] : from_f32<T>(0.f);
        }
      }
    };
    bool more = walk.next(a, s, t);
    if (more) tokens(t), load();
    for (int n = 0; more; ++n) {
      more = walk.next(a, s, t);
      if (more) tokens(t);  // arrives while this tile is split
      const int st = n % a.stages;
      if (n >= a.stages) ok = tc::mbar_wait(&s.x_empty[st], (n / a.stages - 1) & 1, a.status, 11);
      if (!ok) break;
      const uint32_t sx = base + st * X_STAGE;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int row = tid / ROW_PIECES + i * (256 / ROW_PIECES);
        const uint32_t dst = sx + (c >> 3) * 128 * kSlabRow + row * kSlabRow + (((c & 7) ^ (row & 7)) << 4);
        if constexpr (P == 3) {
          uint4 h[3];
          split8(v[i], h);
#pragma unroll
          for (int p = 0; p < 3; ++p)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + p * KS * 128 * kSlabRow), "r"(h[p].x),
                         "r"(h[p].y), "r"(h[p].z), "r"(h[p].w)
                         : "memory");
        } else {
          const uint4 u = *reinterpret_cast<uint4*>(v[i]);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w)
                       : "memory");
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&s.x_full[st]);
      if (more) load();
    }
  } else if (warp < 16) {  // ---- epilogue: a thread a row, half of its columns
    const int half = (warp - 8) >> 2, m = (warp & 3) * 32 + lane, at = m / a.comps, comp = m % a.comps;
    const bool wide = a.wide;
    bool has[kMostChoices];
    int last = -1;
    for (int n = 0; walk.next(a, s, t); ++n) {
      const int buf = n % a.buffers;
      const bool live = at < t.count;
      const int token = live ? a.order[t.place + at] : 0;
      const int64_t row = (int64_t)token * a.comps + comp;
      float f[kMostChoices], dot[kMostChoices];
      if (t.key != last) {
        last = t.key;
#pragma unroll
        for (int j = 0; j < kMostChoices; ++j) has[j] = j < a.per_token && choice(a, last, j) >= 0;
      }
#pragma unroll
      for (int j = 0; j < kMostChoices; ++j) {
        f[j] = has[j] && live ? a.weights[(int64_t)token * a.per_token + j] : 0.f;
        dot[j] = 0.f;
      }
      // after a wait that ran out the warps still meet at the barrier below, for every tile
      ok = ok && tc::mbar_wait(&s.acc_full[buf], (n / a.buffers) & 1, a.status, 13);
      tc::tc_fence_after();
      const uint32_t lanes = s.tmem + ((uint32_t)((warp & 3) * 32) << 16) + buf * a.per_token * COLS;
#pragma unroll 1
      for (int c = half * (NB / 2); ok && c < (half + 1) * (NB / 2) && c < a.features; c += 16) {
        float y[16], xs[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = 0.f;
        if (BACK && a.dots && live)
          load16(static_cast<const T*>(a.x) + row * a.features + c, xs, a.features - c, wide);
        else
#pragma unroll
          for (int i = 0; i < 16; ++i) xs[i] = 0.f;
#pragma unroll
        for (int j = 0; j < kMostChoices; ++j) {
          if (!has[j]) continue;
          uint32_t d[16], w[16];
          __syncwarp();
          tc::tmem_ld16(lanes + j * COLS + c, d);
          if constexpr (P == 3) tc::tmem_ld16(lanes + j * COLS + NB + c, w);
          tc::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float z = __uint_as_float(d[i]);
            if constexpr (P == 3) z += __uint_as_float(w[i]);
            y[i] = fmaf(f[j], z, y[i]);
            if constexpr (BACK) dot[j] = fmaf(z, xs[i], dot[j]);
          }
        }
        if (live && a.out) store16(static_cast<T*>(a.out) + row * a.features + c, y, a.features - c, wide);
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&s.acc_empty[buf]);
      if (BACK && a.dots) {
#pragma unroll
        for (int j = 0; j < kMostChoices; ++j) s.dots[n & 1][half][m][j] = dot[j];
        asm volatile("bar.sync 1, 256;" ::: "memory");  // the other parity's sums were read before the last one
        for (int i = tid - 256; i < t.count * a.per_token; i += 256) {
          const int u = i / a.per_token, j = i % a.per_token;
          float d = 0.f;  // stays zero for a choice without an expert: its rows' products are
          for (int k = u * a.comps; k < (u + 1) * a.comps; ++k) d += s.dots[n & 1][0][k][j] + s.dots[n & 1][1][k][j];
          a.dots[(int64_t)a.order[t.place + u] * a.per_token + j] = d;
        }
      }
    }
  } else if (warp == 16) {  // ---- weights: loaded when the choice changes
    if (lane == 0) {
      int loads = 0, last = -1;
      while (ok && walk.next(a, s, t)) {
        if (t.key == last) continue;
        last = t.key;
        if (loads > 0) ok = tc::mbar_wait(&s.w_empty, (loads - 1) & 1, a.status, 14);
        if (!ok) break;
        int n = 0;
        for (int j = 0; j < a.per_token; ++j) n += choice(a, t.key, j) >= 0;
        tc::mbar_arrive_expect_tx(&s.w_full, n * P * W_PLANE);
        for (int j = 0; j < a.per_token; ++j) {
          const int e = choice(a, t.key, j);
          if (e < 0) continue;
          for (int p = 0; p < P; ++p) {
            const uint32_t dst = wbase + (j * P + p) * W_PLANE;
            if constexpr (BACK) {
              for (int q = 0; q < NB / 64; ++q)
                for (int k = 0; k < KS; ++k)
                  tma_tile4(dst + (q * KS + k) * 64 * kSlabRow, &mw, q * 64, k * 64, e, p, &s.w_full);
            } else {
              for (int k = 0; k < KS; ++k) tma_tile4(dst + k * NB * kSlabRow, &mw, k * 64, 0, e, p, &s.w_full);
            }
          }
        }
        ++loads;
      }
    }
    __syncwarp();
  } else {  // ---- products
    if (lane == 0) {
      const uint32_t idesc = idesc_of<E>((a.features + 15) / 16 * 16, false, BACK);
      const int steps = (a.Kd + 15) / 16;
      int loads = 0;
      bool more = walk.next(a, s, t);
      int last = -1;
      unsigned has = 0;  // bit j: the j-th choice has an expert
      for (int n = 0; more && ok; ++n) {
        const JointTile u = t;
        more = walk.next(a, s, t);
        const int st = n % a.stages, buf = n % a.buffers;
        if (u.key != last) {
          ok = tc::mbar_wait(&s.w_full, loads & 1, a.status, 15);
          ++loads;
          last = u.key;
          has = 0;
          for (int j = 0; j < a.per_token; ++j) has |= (unsigned)(choice(a, last, j) >= 0) << j;
        }
        if (n >= a.buffers) ok = ok && tc::mbar_wait(&s.acc_empty[buf], (n / a.buffers - 1) & 1, a.status, 16);
        ok = ok && tc::mbar_wait(&s.x_full[st], (n / a.stages) & 1, a.status, 17);
        if (!ok) break;
        tc::tc_fence_after();
        const uint32_t sx = base + st * X_STAGE;
        const uint64_t da = desc128(base + st * X_STAGE, 16, 1024);
#pragma unroll
        for (int j = 0; j < kMostChoices; ++j) {
          if (!(has >> j & 1)) continue;
          const uint32_t d = s.tmem + (buf * a.per_token + j) * COLS;
          const uint64_t db = desc128(wbase + j * P * W_PLANE, BACK ? KS * 64 * kSlabRow : 16, 1024);
#pragma unroll
          for (int k = 0; k < 4 * KS; ++k) {
            if (k >= steps) break;
            constexpr int A_PLANE = KS * 128 * kSlabRow;
            const int ka = (k >> 2) * 128 * kSlabRow + (k & 3) * 32;
            const int kb = BACK ? k * 2048 : (k >> 2) * NB * kSlabRow + (k & 3) * 32;
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
              for (int q = 0; q < P; ++q)
                if (p + q < P) {
                  const bool small = P == 3 && p + q > 0;
                  const bool fresh = k == 0 && (small ? p == 0 && q == 1 : true);
                  mma_ss<E>(d + (small ? NB : 0), da + ((p * A_PLANE + ka) >> 4), db + ((q * W_PLANE + kb) >> 4), idesc, !fresh);
                }
          }
        }
        tc::mma_commit(&s.x_empty[st]);
        tc::mma_commit(&s.acc_full[buf]);
        if (more && t.key != u.key) tc::mma_commit(&s.w_empty);
      }
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp == 17) {
    tc::tc_fence_after();
    tc::tmem_dealloc(s.tmem, 512);
  }
}

template <typename T, int NB, int KS, bool BACK>
int launch_joint(const JointArgs& in, const Operand<typename Of<T>::E>& w, cudaStream_t st) {
  using E = typename Of<T>::E;
  constexpr int P = Of<T>::P;
  constexpr int X_STAGE = P * KS * 128 * kSlabRow, W_PLANE = KS * NB * kSlabRow;
  JointArgs a = in;
  a.stages = std::min<int>(kMostStages, (kSmem - a.per_token * P * W_PLANE) / X_STAGE);
  a.buffers = 512 / (a.per_token * NB * (P == 3 ? 2 : 1)) >= 2 ? 2 : 1;
  const int smem = a.stages * X_STAGE + a.per_token * P * W_PLANE + 1024;
  CUtensorMap mw;
  FSC_TRY(tile_map(&mw, w, BACK ? 64 : NB, true));
  auto go = [&](auto kernel) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return check_launch("expert_linear");
    kernel<<<sm_count(), kJointThreads, smem, st>>>(mw, a);
    return check_launch("expert_linear joint");
  };
  return a.Kd % (16 / sizeof(T)) == 0 ? go(joint_kernel<T, E, P, NB, KS, BACK, true>) : go(joint_kernel<T, E, P, NB, KS, BACK, false>);
}

}  // namespace

bool joint_fits(int dtype, int64_t tokens, int64_t per_token, int64_t comps, int64_t experts, int64_t features, int64_t contraction) {
  const int64_t bins = fsc_expert_joint_bins(tokens, per_token, experts);
  if (bins == 0 || per_token > kMostChoices || features > 128 || contraction > 128 || comps > 128) return false;
  const int p = dtype == FSC_F32 ? 3 : 1, nb = features <= 64 ? 64 : 128, ks = contraction <= 64 ? 1 : 2;
  return per_token * nb * (p == 3 ? 2 : 1) <= 512 &&
         per_token * p * ks * nb * kSlabRow + p * ks * 128 * kSlabRow <= kSmem;
}

int joint_product(int dtype, bool back, const JointCall& c, void* workspace, size_t* bytes, cudaStream_t st) {
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    Arena arena(workspace, bytes ? 0 : c.workspace_bytes);
    Operand<typename Of<T>::E> w;
    FSC_TRY(weights_operand(static_cast<const T*>(c.w), c.experts, c.outputs, c.inputs, arena, &w, st));
    if (bytes) {
      *bytes = arena.off;
      return FSC_OK;
    }
    JointArgs a{};
    a.in = c.in, a.x = c.x, a.weights = c.weights, a.offsets = c.offsets, a.order = c.order, a.status = c.status;
    a.out = c.out, a.dots = c.dots;
    a.bins = (int)fsc_expert_joint_bins(c.tokens, c.per_token, c.experts);
    a.experts = (int)c.experts, a.per_token = (int)c.per_token, a.comps = (int)c.comps;
    a.features = (int)(back ? c.inputs : c.outputs), a.Kd = (int)(back ? c.outputs : c.inputs);
    a.per_tile = 128 / a.comps;
    a.wide = a.features % 16 == 0 && (reinterpret_cast<uintptr_t>(c.out) & 31) == 0;
    auto go = [&](auto nb, auto ks) {
      return back ? launch_joint<T, decltype(nb)::value, decltype(ks)::value, true>(a, w, st)
                  : launch_joint<T, decltype(nb)::value, decltype(ks)::value, false>(a, w, st);
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    using N64 = std::integral_constant<int, 64>;
    using N128 = std::integral_constant<int, 128>;
    if (a.features <= 64) return a.Kd <= 64 ? go(N64{}, One{}) : go(N64{}, Two{});
    return a.Kd <= 64 ? go(N128{}, One{}) : go(N128{}, Two{});
  });
}

}  // namespace fsc
