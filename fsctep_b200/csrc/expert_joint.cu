// Experts' products of narrow rows (up to 128 channels), all choices of a token at once.
//
//   out[t, k, :] = sum_j w[t, j] W_j x[t, k, :],  W_j the matrix of the token's j-th choice
//   gradient:  gx[t, k, :] = sum_j w[t, j] W_j^T g[t, k, :],  gw[t, j] = sum_k <W_j^T g[t, k, :], x[t, k, :]>
//
// Bound by memory: at 64 channels a row is 256 bytes and its products 16 kFLOP.  Taken slot by slot a row
// would be read top_k times and its products written and read again; here tokens are grouped by their
// whole choice (the plan's joint grouping), so a tile of 128 rows meets the same few matrices, is read
// once and written once: 50,021 atoms of 9 x 64 fp32 values through 2 of 8 experts take 68 us and the
// gradients 103 us (35 and 53 us of bytes; 1.5 ms in all slot by slot).  What holds it above its bytes is the
// instruction latency of the warps around the products.  A block owns consecutive tiles and keeps the choice's matrices
// in shared memory until the choice changes.  Twelve (gradient: eight) warps load the rows, split them into bfloat16 planes (fp32) and store the
// 128-byte-swizzled operand; one warp issues tcgen05.mma, rows as TMEM lanes, the matrices of all choices
// next to each other as one N (an operand of 128 rows costs its reading from shared memory, 64 bytes a
// cycle, with every product: 96 cycles with 64 columns, 128 with 128); three groups of four warps take the
// finished tiles in turn and join the columns with the token's weights, a row a thread.  The fp32 form adds
// its five small products first and the large one last, so that the running sum, which the tensor
// pipe cuts with every step, is large for Kd / 16 steps only.
#include "expert_joint.cuh"
#include "expert_tc.cuh"

namespace fsc {
namespace {

constexpr int kMostChoices = 4;
constexpr int kMostStages = 2;   // a third left an L1 of a few KB, and the gradient took 167 us instead of 146
constexpr int kSmem = 204800;    // of the matrices and the rows' stages, beside 20 KB of static shared memory
constexpr int kGroups = 3;  // groups of four epilogue warps
// Warps: rows, 12 of the epilogue, weights, products.  The gradient's epilogue also holds rows of x: fewer row
// warps leave it 80 registers instead of 72.
constexpr int row_warps(bool back) { return back ? 8 : 12; }
constexpr int joint_threads(bool back) { return (row_warps(back) + 14) * 32; }

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
  int wide;  // rows of out and x in pieces of 8 values, out on 32 bytes
};

struct JointShared {
  uint64_t x_full[kMostStages], x_empty[kMostStages], w_full, w_empty;
  uint64_t acc_full[kGroups], acc_empty[kGroups];  // of each group's tiles, whatever columns they use
  uint32_t tmem;
  int32_t tiles[1025], first[1025];  // tiles and places before each choice
  float dots[kGroups][2][128][kMostChoices];  // [group][its tile's parity][row][choice]
};

__device__ __forceinline__ void store8(float* p, const float* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// Eight values of a row as T; `whole`: all eight exist and the address is a multiple of 32 (fp32) or 16 bytes.
template <typename T>
__device__ __forceinline__ void store_row8(T* p, const float* v, int n, bool whole) {
  if (whole) {
    if constexpr (sizeof(T) == 4) {
      store8(p, v);
    } else {
      Pack<T, 8> q;
#pragma unroll
      for (int i = 0; i < 8; ++i) q.v[i] = from_f32<T>(v[i]);
      *reinterpret_cast<Pack<T, 8>*>(p) = q;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = from_f32<T>(v[i]);
  }
}
template <typename T>
__device__ __forceinline__ void load_row8(const T* p, float* v, int n, bool whole) {
  if (whole) {
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int b = 0; b < 8; b += E) {
      const Pack<T, E> q = *reinterpret_cast<const Pack<T, E>*>(p + b);
#pragma unroll
      for (int i = 0; i < E; ++i) v[b + i] = to_f32(q.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.f;
  }
}

__device__ __forceinline__ void tmem_ld8(uint32_t at, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(at)
               : "memory");
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
__global__ void __launch_bounds__(joint_threads(BACK), 1) joint_kernel(const __grid_constant__ CUtensorMap mw, JointArgs a) {
  constexpr int X_STAGE = P * KS * 128 * kSlabRow, W_PLANE = KS * NB * kSlabRow;
  constexpr int kRowWarps = row_warps(BACK), kThreads = joint_threads(BACK);
  const int cols = a.per_token * NB;  // TMEM columns of a tile
  extern __shared__ uint8_t dyn[];
  __shared__ JointShared s;
  const uint32_t base = (tc::smem_u32(dyn) + 1023) & ~1023u, wbase = base + a.stages * X_STAGE;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int failed = __ldcg(a.status);
  if (tid == 0) {
    for (int i = 0; i < kMostStages; ++i) tc::mbar_init(&s.x_full[i], kRowWarps), tc::mbar_init(&s.x_empty[i], 1);
    for (int i = 0; i < kGroups; ++i) tc::mbar_init(&s.acc_full[i], 1), tc::mbar_init(&s.acc_empty[i], 4);
    tc::mbar_init(&s.w_full, 1), tc::mbar_init(&s.w_empty, 1);
    tc::fence_mbar_init();
  }
  for (int b = tid; b <= a.bins; b += kThreads) {
    const int here = a.offsets[b];
    s.first[b] = here;
    if (b < a.bins) s.tiles[b + 1] = (a.offsets[b + 1] - here + a.per_tile - 1) / a.per_tile;
  }
  if (warp == kRowWarps + 13) {
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
  bool ok = __all_sync(0xffffffffu, failed == 0);
  if (warp < kRowWarps) {  // ---- rows
    constexpr int THREADS = kRowWarps * 32, ROW_PIECES = 8 * KS, ALL = 128 * ROW_PIECES;
    constexpr int PIECES = (ALL + THREADS - 1) / THREADS;
    int where[PIECES];  // token of the tile and component of each piece's row
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int row = (tid + i * THREADS) / ROW_PIECES;
      where[i] = row / a.comps << 16 | row % a.comps;  // past the last piece: a token that no tile has
    }
    T v[PIECES][8];
    int token[PIECES];
    auto tokens = [&](const JointTile& q, int* tok) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) tok[i] = (where[i] >> 16) < q.count ? a.order[q.place + (where[i] >> 16)] : -1;
    };
    auto load = [&] {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int col = (tid + i * THREADS) % ROW_PIECES * 8;
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
    // A row block's bytes on their way to the L2 a tile before they are read (one thread per token).
    auto prefetch = [&](const void* p, int width, const int* tok) {
      const uint32_t bytes = (uint32_t)a.comps * width * sizeof(T);
      if (bytes % 16 != 0) return;
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        if ((tid + i * THREADS) % ROW_PIECES == 0 && (where[i] & 0xffff) == 0 && tok[i] >= 0)
          asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(static_cast<const T*>(p) +
                                                                        (int64_t)tok[i] * a.comps * width),
                       "r"(bytes)
                       : "memory");
    };
    int coming[PIECES];
    bool more = walk.next(a, s, t), after = false;
    if (more) {
      tokens(t, token);
      load();
      if (BACK && a.dots) prefetch(a.x, a.features, token);
      after = walk.next(a, s, t);
      if (after) tokens(t, coming);
    }
    for (int n = 0; more; ++n) {
      more = after;
      if (more) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) token[i] = coming[i];
        prefetch(a.in, a.Kd, token);
        if (BACK && a.dots) prefetch(a.x, a.features, token);
        after = walk.next(a, s, t);
        if (after) tokens(t, coming);
      }
      const int st = n % a.stages;
      if (n >= a.stages) ok = wait_warp(&s.x_empty[st], (n / a.stages - 1) & 1, a.status, 11);
      if (!ok) break;
      const uint32_t sx = base + st * X_STAGE;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int q = tid + i * THREADS, row = q / ROW_PIECES, c = q % ROW_PIECES;
        if (q >= ALL) continue;
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
  } else if (warp < kRowWarps + 12) {  // ---- epilogue: a thread a row; group g takes every third tile
    const int g = (warp - kRowWarps) >> 2, m = (warp & 3) * 32 + lane, at = m / a.comps, comp = m % a.comps;
    const bool wide = a.wide;
    bool has[kMostChoices];
    int last = -1;
    JointTile u;
    int token = 0;
    float f[kMostChoices];
    // the next tile of this group, its token and weights: on their way while the last one is joined
    auto fetch = [&](JointTile& q) -> bool {
      if (!walk.next(a, s, q)) return false;
      token = at < q.count ? a.order[q.place + at] : -1;
#pragma unroll
      for (int j = 0; j < kMostChoices; ++j)
        f[j] = token >= 0 && j < a.per_token ? a.weights[(int64_t)token * a.per_token + j] : 0.f;
      return true;
    };
    bool more = true;
    for (int i = 0; i < g && more; ++i) more = walk.next(a, s, u);
    more = more && fetch(u);
    for (int n = g; more; n += kGroups) {
      t = u;
      const int mine = token, buf = n % a.buffers;
      float w[kMostChoices], dot[kMostChoices];
      if (t.key != last) {
        last = t.key;
#pragma unroll
        for (int j = 0; j < kMostChoices; ++j) has[j] = j < a.per_token && choice(a, last, j) >= 0;
      }
#pragma unroll
      for (int j = 0; j < kMostChoices; ++j) w[j] = has[j] ? f[j] : 0.f, dot[j] = 0.f;
      more = true;
      for (int i = 1; i < kGroups && more; ++i) more = walk.next(a, s, u);
      more = more && fetch(u);
      const int64_t row = (int64_t)mine * a.comps + comp;
      const bool want = BACK && a.dots && mine >= 0;
      const T* x = static_cast<const T*>(a.x) + row * a.features;
      float xs[2][8];  // eight columns of x each, loaded two steps before their use
      if (want) {
        load_row8(x, xs[0], a.features, wide);
        if (a.features > 8) load_row8(x + 8, xs[1], a.features - 8, wide);
      }
      // after a wait that ran out the warps still meet at the barrier below, for every tile
      ok = ok && wait_warp(&s.acc_full[g], (n / kGroups) & 1, a.status, 13);
      tc::tc_fence_after();
      const uint32_t lanes = s.tmem + ((uint32_t)((warp & 3) * 32) << 16) + buf * cols;
      T* out = static_cast<T*>(a.out) + row * a.features;
#pragma unroll 1
      for (int c0 = 0; ok && c0 < a.features; c0 += 16)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = c0 + 8 * h;
          if (c >= a.features) break;
          float y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = 0.f;
#pragma unroll
          for (int j0 = 0; j0 < kMostChoices; j0 += 2) {
            if (j0 >= a.per_token) break;
            uint32_t d[2][8];
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (has[j0 + j]) tmem_ld8(lanes + (j0 + j) * NB + c, d[j]);
            tc::tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (has[j0 + j])
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const float z = __uint_as_float(d[j][i]);
                  y[i] = fmaf(w[j0 + j], z, y[i]);
                  if constexpr (BACK) dot[j0 + j] = fmaf(z, xs[h][i], dot[j0 + j]);  // not used without `want`
                }
          }
          if (want && c + 16 < a.features) load_row8(x + c + 16, xs[h], a.features - c - 16, wide);
          if (mine >= 0 && a.out) store_row8(out + c, y, a.features - c, wide);
        }
      if (!ok) {
        const float y[8] = {failed_value(), failed_value(), failed_value(), failed_value(),
                            failed_value(), failed_value(), failed_value(), failed_value()};
        for (int c = 0; mine >= 0 && a.out && c < a.features; c += 8) store_row8(out + c, y, a.features - c, wide);
#pragma unroll
        for (int j = 0; j < kMostChoices; ++j) dot[j] = failed_value();
      }
      tc::tc_fence_before();
      __syncwarp();
      if (ok && lane == 0) tc::mbar_arrive(&s.acc_empty[g]);
      if (BACK && a.dots) {
        float(*sums)[kMostChoices] = s.dots[g][(n / kGroups) & 1];
#pragma unroll
        for (int j = 0; j < kMostChoices; ++j) sums[m][j] = want && has[j] ? dot[j] : 0.f;
        // the group's four warps; the other parity's sums were read before the last barrier
        if (g == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
        else if (g == 1) asm volatile("bar.sync 2, 128;" ::: "memory");
        else asm volatile("bar.sync 3, 128;" ::: "memory");
        for (int i = (warp & 3) * 32 + lane; i < t.count * a.per_token; i += 128) {
          const int v = i / a.per_token, j = i % a.per_token;
          float d = 0.f;  // stays zero for a choice without an expert: its rows' products are
          for (int k = v * a.comps; k < (v + 1) * a.comps; ++k) d += sums[k][j];
          a.dots[(int64_t)a.order[t.place + v] * a.per_token + j] = d;
        }
      }
    }
  } else if (warp == kRowWarps + 12) {  // ---- weights: loaded when the choice changes
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
            const uint32_t dst = wbase + p * a.per_token * W_PLANE;
            for (int k = 0; k < KS; ++k) {
              if constexpr (BACK) {
                for (int q = 0; q < NB / 64; ++q)
                  tma_tile4(1, dst + ((j * (NB / 64) + q) * KS + k) * 64 * kSlabRow, &mw, q * 64, k * 64, e, p, tc::smem_u32(&s.w_full));
              } else {
                tma_tile4(1, dst + (k * a.per_token + j) * NB * kSlabRow, &mw, k * 64, 0, e, p, tc::smem_u32(&s.w_full));
              }
            }
          }
        }
        ++loads;
      }
      if (!ok && loads > 0) drain(&s.w_full, (loads - 1) & 1);
    }
    __syncwarp();
  } else {  // ---- products
    const uint32_t issue = elect_one(), tmem = __shfl_sync(0xffffffffu, s.tmem, 0);
    const int steps = (a.Kd + 15) / 16;
    int loads = 0, last = -1, count = 0, n = 0;
    bool more = walk.next(a, s, t);
    for (; more && ok; ++n) {
      const JointTile u = t;
      more = walk.next(a, s, t);
      const int st = n % a.stages, buf = n % a.buffers;
      if (u.key != last) {
        ok = wait_warp(&s.w_full, loads & 1, a.status, 15);
        ++loads;
        last = u.key;
        count = 0;  // choices up to the last that has an expert; what the others' columns hold is not read
        for (int j = 0; j < a.per_token; ++j)
          if (choice(a, last, j) >= 0) count = j + 1;
      }
      const int before = n - a.buffers;  // the tile that used these columns last
      if (before >= 0) ok = ok && wait_warp(&s.acc_empty[before % kGroups], (before / kGroups) & 1, a.status, 16);
      ok = ok && wait_warp(&s.x_full[st], (n / a.stages) & 1, a.status, 17);
      if (!ok) break;
      tc::tc_fence_after();
      if (count > 0) {
        const uint32_t idesc = idesc_of<E>(count * NB, false, BACK), d = tmem + buf * cols;
        const uint64_t da = desc128(base + st * X_STAGE, 16, 1024);
        const uint64_t db = desc128(wbase, BACK ? KS * 64 * kSlabRow : 16, 1024);
        bool fresh = true;
#pragma unroll
        for (int large = P == 3 ? 0 : 1; large < 2; ++large)  // planes are 2^-8 apart: products down to 2^-16
#pragma unroll
          for (int k = 0; k < 4 * KS; ++k) {
            if (k >= steps) break;
            const int ka = (k >> 2) * 128 * kSlabRow + (k & 3) * 32;
            const int kb = BACK ? k * 2048 : (k >> 2) * cols * kSlabRow + (k & 3) * 32;
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
              for (int q = 0; q < P; ++q)
                if (p + q < P && (p + q == 0) == (large == 1)) {
                  mma_ss<E>(issue, d, da + ((p * KS * 128 * kSlabRow + ka) >> 4), db + ((q * a.per_token * W_PLANE + kb) >> 4),
                            idesc, !fresh);
                  fresh = false;
                }
          }
      }
      commit_if(issue, &s.x_empty[st]);
      commit_if(issue, &s.acc_full[n % kGroups]);
      if (more && t.key != u.key) commit_if(issue, &s.w_empty);
    }
    if (!ok && n > 0) drain(&s.x_empty[(n - 1) % a.stages], ((n - 1) / a.stages) & 1);
    __syncwarp();
  }
  __syncthreads();
  if (warp == kRowWarps + 13) {
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
  a.buffers = std::min(kGroups, 512 / (a.per_token * NB));
  const int smem = a.stages * X_STAGE + a.per_token * P * W_PLANE + 1024;
  CUtensorMap mw;
  FSC_TRY(tile_map(&mw, w, BACK ? 64 : NB, true));
  auto go = [&](auto kernel) {
    if (!allow_shared(kernel, kSmem + 1024)) return check_launch("expert_linear");
    kernel<<<sm_count(), joint_threads(BACK), smem, st>>>(mw, a);
    return check_launch("expert_linear joint");
  };
  return a.Kd % (16 / sizeof(T)) == 0 ? go(joint_kernel<T, E, P, NB, KS, BACK, true>) : go(joint_kernel<T, E, P, NB, KS, BACK, false>);
}

}  // namespace

bool joint_fits(int dtype, int64_t tokens, int64_t per_token, int64_t comps, int64_t experts, int64_t features, int64_t contraction) {
  const int64_t bins = fsc_expert_joint_bins(tokens, per_token, experts);
  if (bins == 0 || per_token > kMostChoices || features > 128 || contraction > 128 || comps > 128) return false;
  const int p = dtype == FSC_F32 ? 3 : 1, nb = features <= 64 ? 64 : 128, ks = contraction <= 64 ? 1 : 2;
  return per_token * nb <= 256 &&
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
    a.wide = a.features % 8 == 0 && (reinterpret_cast<uintptr_t>(c.out) & 31) == 0;
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
