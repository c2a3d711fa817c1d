// Products of rows with the weights of the experts they were routed to, and their gradients.
//
//   rows:   z[slot, k, :] = W_e x[row(slot), k, :]        (or W_e^T g for the gradient in x)
//   weight: dW[e] = sum over e's rows of g (w_slot x)^T
//   join:   out[t, k, :] = sum_j w[t, j] z[(t, j), k, :], and the products <z, x> that the routing
//           weights' gradient needs, in slot order
//
// Bound by the tensor pipe and the L2 for wide layers and many rows, by reading the experts' weights for
// few rows.  A pass copies the rows into the plan's order (each expert's rows next to each other, on a
// multiple of 16), so that everything reaches shared memory as TMA tiles: gathering inside the product
// (TMA gather4, 40 cycles an instruction of four 128-byte rows) kept the tensor pipe at a fifth.  A
// persistent block per SM takes tiles of 128 features by up to NT rows of one expert: the features are the
// M index of tcgen05.mma, so that consecutive TMEM lanes are consecutive addresses of the output and
// every store is coalesced, and the rows are its N index, cut into equal parts of a multiple of 16, so
// that an expert with 225 rows costs 240, not 256 (or 384 in tiles of 128).  Slabs are 128-byte
// swizzled (64 two-byte elements a row) and serve an operand whose rows are its M or N index (K-major) as
// well as one whose rows are the contraction index (MN-major), so nothing is transposed; the weights'
// tensor has the expert as an index of its own, which keeps a ragged edge from reading the next
// expert.  One thread issues the copies, one the products, eight warps read finished accumulators
// while the next are computed (two TMEM buffers).  16-bit and 8-bit operands with more than 128 features take
// tiles of 256 x 256 in pairs of blocks (cta_group::2: a block's multiplier reads half of the rows from its partner).
// 16,384 bf16 rows through 1024 x 2048 experts: 67 us (1.03 PFLOP/s), gradients 65 us in x and
// 123 us in W (76 us without routing weights, whose products with the rows take two operands).
//   32 bits: an element is the sum of three bfloat16 (8 + 8 + 8 significand bits), split by a pass over
//   the operands; the six products down to 2^-16 of the leading one count, the rest is below 2^-21 and 2^-24 on average.
//   8 bits: e4m3 operands, the row's and the output's scale multiply the accumulator.
// The tensor pipe cuts, not rounds, its running sum (about 3e-8 of it for each of Kd / 16 steps).
// Where that shows in the result (32-bit outputs, sums over many rows), a TMEM accumulator runs for
// 256 or 512 elements only and is then added to registers (PROMOTE), and the five small products of the
// 32-bit form have an accumulator of their own.
#include "expert_joint.cuh"
#include "expert_tc.cuh"

namespace fsc {
namespace {

constexpr int kThreads = 320;  // warps 0-7 epilogue, 8 copies, 9 products
constexpr int BM = 128;        // features of a tile
// Slabs (of 64 elements) of one accumulator under PROMOTE: 16 steps of the cut sum in 32 bits (about 2e-7), 32 in 16 bits
// (4e-7; up to 96 in the weighted weight gradient, 1e-6).
template <int P>
constexpr int group_of = P == 3 ? 4 : 8;

struct ProductArgs {
  const float* row_weight;  // per slot factor, or null
  const float* x_scale;     // 8 bits: per row of x
  const float* w_scale;     // 8 bits: [experts][M]
  const int32_t* offsets;
  const int32_t* order;
  int32_t* status;
  void* out;
  int experts, per_token, comps;  // per_token: slots of a token
  int x_by_slot;                  // 8 bits: x_scale has a value for each slot, not for each token
  int M, N, Kd;                   // rows: features out, -, contraction; weight: inputs, outputs, -
  int tiles_m, tiles_n, splits;
};

// PA, PB: planes of the operands; NT: rows (or outputs) of a tile; of a pair's tile each block keeps half.
template <int PA, int PB, int NT, bool PAIR>
struct Shape {
  static constexpr int MINE = PAIR ? NT / 2 : NT;
  static constexpr int A_BYTES = PA * BM * kSlabRow, B_BYTES = PB * MINE * kSlabRow;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = 196608 / STAGE;
  static constexpr int SMEM = STAGES * STAGE + 1024;
};

// Where each expert's rows start in plan order: multiples of 16.  One warp.
template <int NT>
__device__ __forceinline__ void scan_experts(const int32_t* offsets, int experts, int comps, int32_t* base, int32_t* tiles) {
  const int lane = threadIdx.x & 31;
  int rows_before = 0, tiles_before = 0;
  for (int e0 = 0; e0 < experts; e0 += 32) {
    const int e = e0 + lane;
    const int n = e < experts ? (offsets[e + 1] - offsets[e]) * comps : 0;
    const int r = (n + 15) & ~15, t = (n + NT - 1) / NT;
    int x = r, y = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) x += u, y += v;
    }
    if (e < experts) {
      base[e] = rows_before + x - r;
      if (tiles) tiles[e] = tiles_before + y - t;
    }
    rows_before += __shfl_sync(0xffffffffu, x, 31);
    tiles_before += __shfl_sync(0xffffffffu, y, 31);
  }
  if (lane == 0) {
    base[experts] = rows_before;
    if (tiles) tiles[experts] = tiles_before;
  }
}

struct Shared {
  uint64_t full[6], empty[6], acc_full[2], acc_empty[2];
  uint32_t tmem;
  int32_t base[1025];   // first sorted row of an expert
  int32_t tiles[1025];  // rows product: row tiles of the experts before
  alignas(16) int2 rows[8][128];  // of each epilogue warp's columns: output row, factor (the bits of a float)
};

struct Tile {
  int e, m0, n0, count;  // count: rows (rows product) or outputs (weight product) of the tile
  int place;             // rows product: first place of the tile in the plan's order, times comps
  int row, rows, nk;     // first sorted row; weight product: the rows that it sums; stages
  int split;
};

template <bool DW, int NT, int KC, int WIDE_M>
__device__ __forceinline__ bool tile_of(const ProductArgs& a, const Shared& s, int id, Tile& t) {
  if constexpr (DW) {
    if (id >= a.experts * a.tiles_m * a.tiles_n * a.splits) return false;
    t.m0 = (id % a.tiles_m) * WIDE_M;
    id /= a.tiles_m;
    t.n0 = (id % a.tiles_n) * NT;
    id /= a.tiles_n;
    t.split = id % a.splits;
    t.e = id / a.splits;
    t.count = min(NT, a.N - t.n0);
    const int rows = s.base[t.e + 1] - s.base[t.e];  // the ones that fill up to 16 are zero
    const int part = ((rows + a.splits - 1) / a.splits + 63) / 64 * 64;
    const int lo = min(t.split * part, rows);
    t.row = s.base[t.e] + lo;
    t.rows = min(part, rows - lo);
    t.nk = (t.rows + 63) / 64;
    t.place = 0;
  } else {
    const int rt = id / a.tiles_m;
    if (rt >= s.tiles[a.experts]) return false;
    t.e = find_expert(s.tiles, a.experts, rt);
    const int first = a.offsets[t.e] * a.comps, rows = a.offsets[t.e + 1] * a.comps - first;
    const int parts = s.tiles[t.e + 1] - s.tiles[t.e];
    const int per = ((rows + parts - 1) / parts + 15) / 16 * 16;
    const int at = (rt - s.tiles[t.e]) * per;
    t.m0 = (id % a.tiles_m) * WIDE_M;
    t.n0 = 0;
    t.count = min(per, rows - at);
    t.place = first + at;
    t.row = s.base[t.e] + at;
    t.rows = t.count;
    t.nk = (a.Kd + KC - 1) / KC;
    t.split = 0;
  }
  return true;
}

// T: element of the operands (e4m3, half, bfloat16), PA, PB: their planes; A_MN: the weights' rows are the contraction
// index (W^T); DW: the weight product (A: the scaled rows of x, B: the rows of g); PAIR: two blocks share a tile of
// 256 features, each with its 128 features and half of the rows in shared memory and all rows of its features in TMEM.
template <typename T, int PA, int PB, int NT, bool A_MN, bool DW, bool PROMOTE, bool PAIR, typename OUT>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb, ProductArgs a) {
  using S = Shape<PA, PB, NT, PAIR>;
  constexpr int KE = kSlabRow / sizeof(T);  // elements of a slab row
  constexpr int KC = DW ? 64 : KE;          // contraction of a stage
  constexpr int HALF = NT / 2;              // columns of an epilogue warp
  constexpr int WIDE_M = PAIR ? 2 * BM : BM;
  constexpr int kGroup = group_of<PA>;
  constexpr int STEP_N = PAIR ? 32 : 16;    // a product's N is a multiple of this
  extern __shared__ uint8_t dyn[];
  __shared__ Shared s;
  const uint32_t base = (tc::smem_u32(dyn) + 1023) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = PAIR ? (int)cluster_rank() : 0;
  const int unit = PAIR ? blockIdx.x / 2 : blockIdx.x, units = PAIR ? gridDim.x / 2 : gridDim.x;
  const int failed = __ldcg(a.status);
  if (tid == 0) {
    for (int i = 0; i < S::STAGES; ++i) tc::mbar_init(&s.full[i], 1), tc::mbar_init(&s.empty[i], 1);
    for (int i = 0; i < 2; ++i) tc::mbar_init(&s.acc_full[i], 1), tc::mbar_init(&s.acc_empty[i], PAIR ? 16 : 8);
    tc::fence_mbar_init();
  }
  if (warp == 9) tmem_take<PAIR>(&s.tmem);
  if (warp == 8) scan_experts<NT>(a.offsets, a.experts, a.comps, s.base, s.tiles);
  tc::tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // the partner's barriers exist
  tc::tc_fence_after();
  auto tile = [&](int id, Tile& t) { return tile_of<DW, NT, KC, WIDE_M>(a, s, id, t); };
  auto wide_n = [&](const Tile& t) { return DW && PAIR ? NT : (t.count + STEP_N - 1) / STEP_N * STEP_N; };
  Tile t;
  bool ok = __all_sync(0xffffffffu, failed == 0);
  int kt = 0;  // stages so far
  if (warp < 8) {  // ---- epilogue: lane = feature, column = row (or output)
    const int c0 = (warp >> 2) * HALF;
    int group = 0;
    auto release = [&](int buf) {  // the columns may be written again: the products are issued by the first block
      if constexpr (PAIR) arrive_cluster(in_first_block(tc::smem_u32(&s.acc_empty[buf])));
      else tc::mbar_arrive(&s.acc_empty[buf]);
    };
    for (int id = unit; tile(id, t); id += units) {
      const int m = t.m0 + rank * BM + (warp & 3) * 32 + lane;
      const int groups = PROMOTE ? (t.nk + kGroup - 1) / kGroup : 1;
      if constexpr (!DW) {  // where this warp's columns go, before their sums are there
        __syncwarp();
#pragma unroll
        for (int i = 0; i < HALF / 32; ++i) {
          int2 where = make_int2(0, 0);
          if (c0 + i * 32 + lane < t.count) {
            const int r = t.place + c0 + i * 32 + lane, slot = a.order[r / a.comps];
            float f = a.row_weight ? a.row_weight[slot] : 1.f;
            if constexpr (sizeof(T) == 1) f *= a.x_scale[a.x_by_slot ? slot : slot / a.per_token];
            where = make_int2(slot * a.comps + r % a.comps, __float_as_int(f));
          }
          s.rows[warp][i * 32 + lane] = where;
        }
        __syncwarp();
      }
      float acc[PROMOTE ? HALF : 1];
      if constexpr (PROMOTE) {
#pragma unroll
        for (int i = 0; i < HALF; ++i) acc[i] = 0.f;
        for (int g = 0; g < groups; ++g, ++group) {
          const int buf = group & 1;
          ok = ok && wait_warp(&s.acc_full[buf], (group >> 1) & 1, a.status, 3);
          if (!ok) break;
          tc::tc_fence_after();
          const uint32_t at = s.tmem + ((uint32_t)((warp & 3) * 32) << 16) + buf * 256 + c0;
#pragma unroll
          for (int cb = 0; cb < HALF / 16; ++cb) {
            if (c0 + cb * 16 < t.count) {
              uint32_t v[16];
              __syncwarp();
              tc::tmem_ld16(at + cb * 16, v);
              if constexpr (PA == 3) {
                uint32_t w[16];
                tc::tmem_ld16(at + NT + cb * 16, w);
                tc::tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[cb * 16 + i] += __uint_as_float(v[i]) + __uint_as_float(w[i]);
              } else {
                tc::tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[cb * 16 + i] += __uint_as_float(v[i]);
              }
            }
          }
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) release(buf);
        }
        if (!ok) {
#pragma unroll
          for (int i = 0; i < HALF; ++i) acc[i] = failed_value();
        }
      } else {
        ok = ok && wait_warp(&s.acc_full[group & 1], (group >> 1) & 1, a.status, 3);
        tc::tc_fence_after();
      }
      float ws = 1.f;
      if constexpr (sizeof(T) == 1) ws = m < a.M ? a.w_scale[(int64_t)t.e * a.M + m] : 0.f;
      OUT* out = static_cast<OUT*>(a.out);
#pragma unroll
      for (int cb = 0; cb < HALF / 32; ++cb) {
        const int c = c0 + cb * 32;
        if (c >= t.count) continue;  // the whole warp alike
        uint32_t v[32];
        if constexpr (PROMOTE) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(acc[cb * 32 + i]);
        } else {
          __syncwarp();
          if (ok) {
            tc::tmem_ld32(s.tmem + ((uint32_t)((warp & 3) * 32) << 16) + (group & 1) * 256 + c, v);
            tc::tmem_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(failed_value());
          }
        }
        if constexpr (DW) {
          if (m < a.M) {
            OUT* o = out + (((int64_t)t.split * a.experts + t.e) * a.N + t.n0 + c) * a.M + m;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c + j < t.count) o[(int64_t)j * a.M] = from_f32<OUT>(__uint_as_float(v[j]));
          }
        } else {
          const int left = t.count - c;  // rows of this chunk: the whole warp alike
          if (m < a.M) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              // two rows at a time from shared memory: shuffles, one after the other, took 95 cycles a row
              const int4 r = *reinterpret_cast<const int4*>(&s.rows[warp][cb * 32 + j]);
              float y0 = __uint_as_float(v[j]) * __int_as_float(r.y), y1 = __uint_as_float(v[j + 1]) * __int_as_float(r.w);
              if constexpr (sizeof(T) == 1) y0 *= ws, y1 *= ws;
              if (j < left) out[(int64_t)r.x * a.M + m] = from_f32<OUT>(y0);
              if (j + 1 < left) out[(int64_t)r.z * a.M + m] = from_f32<OUT>(y1);
            }
          }
        }
      }
      if constexpr (!PROMOTE) {
        tc::tc_fence_before();
        __syncwarp();
        if (ok && lane == 0) release(group & 1);
        ++group;
      }
    }
  } else if (warp == 8) {  // ---- copies (the warp converged, one lane issuing)
    const uint32_t issue = elect_one();
    for (int id = unit; ok && tile(id, t); id += units) {
      const int n = wide_n(t), mine = PAIR ? n / 2 : n;  // columns of the product, and of them in this block
      const int slabs = (mine + 63) / 64;
      const int e = __shfl_sync(0xffffffffu, t.e, 0), m0 = __shfl_sync(0xffffffffu, t.m0 + rank * BM, 0);
      // rows product: first row of this block's share; weight product: first row, and first output of the share
      const int row = __shfl_sync(0xffffffffu, DW ? t.row : t.row + rank * mine, 0);
      const int n0 = __shfl_sync(0xffffffffu, t.n0 + rank * mine, 0);
      const uint32_t bytes = (PAIR ? 2 : 1) * (S::A_BYTES + PB * slabs * 64 * kSlabRow);
      for (int kc = 0; kc < t.nk; ++kc, ++kt) {
        const int st = kt % S::STAGES;
        if (kt >= S::STAGES) ok = wait_warp(&s.empty[st], (kt / S::STAGES - 1) & 1, a.status, 2);
        if (!ok) break;
        uint32_t bar = tc::smem_u32(&s.full[st]);
        if (rank == 0) expect_if(issue, &s.full[st], bytes);
        if constexpr (PAIR) bar = in_first_block(bar);
        const uint32_t sa = base + st * S::STAGE, sb = sa + S::A_BYTES;
#pragma unroll
        for (int p = 0; p < PA; ++p) {
          const uint32_t pa = sa + p * BM * kSlabRow;
          if constexpr (DW) {
            tma_tile3<PAIR>(issue, pa, &ma, m0, row + kc * 64, p, bar);
            tma_tile3<PAIR>(issue, pa + 64 * kSlabRow, &ma, m0 + 64, row + kc * 64, p, bar);
          } else if constexpr (A_MN) {
            tma_tile4<PAIR>(issue, pa, &ma, m0, kc * KC, e, p, bar);
            tma_tile4<PAIR>(issue, pa + 64 * kSlabRow, &ma, m0 + 64, kc * KC, e, p, bar);
          } else {
            tma_tile4<PAIR>(issue, pa, &ma, kc * KC, m0, e, p, bar);
          }
        }
#pragma unroll
        for (int p = 0; p < PB; ++p) {
          const uint32_t pb = sb + p * S::MINE * kSlabRow;
#pragma unroll
          for (int q = 0; q < S::MINE / 64; ++q)
            if (q < slabs) {
              if constexpr (DW) tma_tile3<PAIR>(issue, pb + q * 64 * kSlabRow, &mb, n0 + q * 64, row + kc * 64, p, bar);
              else tma_tile3<PAIR>(issue, pb + q * 64 * kSlabRow, &mb, kc * KC, row + q * 64, p, bar);
            }
        }
        __syncwarp();
      }
    }
    if (!ok && kt > 0) {  // of a pair all copies arrive in the first block
      bool done = rank == 0;
      for (int i = max(0, kt - S::STAGES); done && i < kt; ++i) done = drain(&s.full[i % S::STAGES], (i / S::STAGES) & 1);
      if (rank != 0) drain_time();
    }
    __syncwarp();
  } else {  // ---- products
    if (rank == 0) {
      const uint32_t issue = elect_one(), tmem = __shfl_sync(0xffffffffu, s.tmem, 0);
      constexpr bool AM = A_MN || DW, BMN = DW;
      constexpr uint32_t A_STEP = AM ? 2048 : 32, B_STEP = BMN ? 2048 : 32, LBO = 64 * kSlabRow;
      int group = 0;
      for (int id = unit; ok && tile(id, t); id += units) {
        const uint32_t idesc = idesc_of<T>(wide_n(t), AM, BMN, WIDE_M);
        uint32_t d = 0;
        for (int kc = 0; kc < t.nk; ++kc, ++kt) {
          const bool first = PROMOTE ? kc % kGroup == 0 : kc == 0;
          const bool last = kc + 1 == t.nk || (PROMOTE && kc % kGroup == kGroup - 1);
          if (first) {
            const int buf = group & 1;
            if (group >= 2) ok = wait_warp(&s.acc_empty[buf], ((group >> 1) - 1) & 1, a.status, 4);
            if (!ok) break;
            d = tmem + buf * 256;
          }
          const int st = kt % S::STAGES;
          ok = wait_warp(&s.full[st], (kt / S::STAGES) & 1, a.status, 1);
          if (!ok) break;
          tc::tc_fence_after();
          const uint32_t sa = base + st * S::STAGE, sb = sa + S::A_BYTES;
          // sorted rows come in sixteens: past the part's last sixteen lie another's
          const int steps = DW ? min(4, (t.rows - kc * 64) / 16) : 4;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < steps)
#pragma unroll
              for (int p = 0; p < PA; ++p)
#pragma unroll
                for (int q = 0; q < PB; ++q)
                  if (p + q < (PA > PB ? PA : PB)) {  // planes are 2^-8 apart: of three each down to 2^-16, of two to 2^-8
                    const bool small = PA == 3 && p + q > 0;
                    const bool fresh = first && k == 0 && (small ? p == 0 && q == 1 : p + q == 0);
                    mma_ss<T, PAIR>(issue, d + (small ? NT : 0),
                                    desc128(sa + p * BM * kSlabRow + k * A_STEP, AM ? LBO : 16, 1024),
                                    desc128(sb + q * S::MINE * kSlabRow + k * B_STEP, BMN ? LBO : 16, 1024), idesc, !fresh);
                  }
          commit_if<PAIR>(issue, &s.empty[st]);
          if (last) {
            commit_if<PAIR>(issue, &s.acc_full[group & 1]);
            ++group;
          }
        }
      }
      if (!ok && kt > 0) drain(&s.empty[(kt - 1) % S::STAGES], ((kt - 1) / S::STAGES) & 1);
    }
    __syncwarp();
  }
  tc::tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // nothing of the pair is in flight
  if (warp == 9) {
    tc::tc_fence_after();
    tmem_give<PAIR>(s.tmem);
  }
}

struct SortArgs {
  const void* in;
  void* out;
  const float* weights;  // slot factors, or null
  const int32_t* offsets;
  const int32_t* order;
  int experts, per_token, comps, by_slot;
  int cols, pitch;
  int64_t out_rows;  // of a plane
};

// Rows in the plan's order, each expert's on a multiple of 16 with zero rows in between.  A warp a row.
template <typename T, typename E, int P, bool VEC>
__global__ void __launch_bounds__(256) sort_kernel(SortArgs a) {
  __shared__ int32_t base[1025];
  if (threadIdx.x < 32) scan_experts<16>(a.offsets, a.experts, a.comps, base, nullptr);
  __syncthreads();
  const int lane = threadIdx.x & 31, rows = base[a.experts];
  constexpr int N = 16 / sizeof(E), U = VEC ? 4 : 1;
  for (int r = blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.x * 8) {
    const int e = find_expert(base, a.experts, r), at = r - base[e], first = a.offsets[e];
    const bool live = at < (a.offsets[e + 1] - first) * a.comps;
    const T* row = static_cast<const T*>(a.in);
    float f = 1.f;
    if (live) {
      const int slot = a.order[first + at / a.comps];
      row += ((int64_t)(a.by_slot ? slot : slot / a.per_token) * a.comps + at % a.comps) * a.cols;
      if (a.weights) f = a.weights[slot];
    }
    E* out = static_cast<E*>(a.out) + (int64_t)r * a.pitch;
    for (int c0 = lane * N; c0 < a.pitch; c0 += 32 * N * U) {
      Piece<T, E, P, VEC> p[U];  // asked for together
#pragma unroll
      for (int u = 0; u < U; ++u) p[u].load(row, live, c0 + u * 32 * N, a.cols);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + u * 32 * N < a.pitch) p[u].store(a.weights != nullptr, f, out + c0 + u * 32 * N, a.out_rows * a.pitch);
    }
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

// NW warps share a token; a block is one token's, or eight warps of one each.  Bound by memory (z read once): a thread
// asks for all of its slots' values of four columns (up to eight slots) before it adds the first.
template <typename T, int NW, int S, int VE>
__global__ void __launch_bounds__(NW == 1 ? 256 : NW * 32) join_kernel(JoinArgs a) {
  constexpr int TPT = NW * 32, Q = S < 8 ? S : 8, PER = NW == 1 ? 8 : 1;
  __shared__ float part[NW][S];
  const int t = threadIdx.x % TPT;
  const int64_t token = (int64_t)blockIdx.x * PER + threadIdx.x / TPT;
  if (token >= a.tokens) return;
  const int64_t slot0 = token * a.per_token;
  float f[S], dot[S];
  unsigned live = 0;
#pragma unroll
  for (int j = 0; j < S; ++j) {
    f[j] = 0.f, dot[j] = 0.f;
    if (j < a.per_token) {
      const int e = a.indices[slot0 + j];
      if (e >= 0 && e < a.experts) {
        live |= 1u << j;
        f[j] = a.weights ? a.weights[slot0 + j] : 1.f;
      }
    }
  }
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
    for (int j0 = 0; j0 < S; j0 += Q) {
      if (j0 >= a.per_token) break;
      alignas(16) float z[Q][VE];
#pragma unroll
      for (int j = 0; j < Q; ++j)
        if (live >> (j0 + j) & 1) {
          // in pieces of 16 bytes: z starts on no more than that
          constexpr int L = VE < 4 ? VE : 4;
          const float* from = a.z + (slot0 + j0 + j) * a.width + c;
#pragma unroll
          for (int i = 0; i < VE; i += L)
            *reinterpret_cast<Pack<float, L>*>(&z[j][i]) = *reinterpret_cast<const Pack<float, L>*>(from + i);
        }
#pragma unroll
      for (int j = 0; j < Q; ++j) {
        if (j0 + j >= a.per_token) continue;
        const bool here = live >> (j0 + j) & 1;
        const int64_t at = (slot0 + j0 + j) * a.width + c;
        if (here && a.x) {
          if (a.x_by_slot) {
            const Pack<T, VE> p = *reinterpret_cast<const Pack<T, VE>*>(static_cast<const T*>(a.x) + at);
#pragma unroll
            for (int i = 0; i < VE; ++i) xs[i] = to_f32(p.v[i]);
          }
#pragma unroll
          for (int i = 0; i < VE; ++i) dot[j0 + j] = fmaf(z[j][i], xs[i], dot[j0 + j]);
        }
        if (a.slot_out) {
          Pack<T, VE> p;
#pragma unroll
          for (int i = 0; i < VE; ++i) p.v[i] = from_f32<T>(here ? z[j][i] * f[j0 + j] : 0.f);
          *reinterpret_cast<Pack<T, VE>*>(static_cast<T*>(a.slot_out) + at) = p;
        }
        if (here) {
#pragma unroll
          for (int i = 0; i < VE; ++i) sum[i] = fmaf(z[j][i], f[j0 + j], sum[i]);
        }
      }
    }
    if (a.out) {
      Pack<T, VE> p;
#pragma unroll
      for (int i = 0; i < VE; ++i) p.v[i] = from_f32<T>(sum[i]);
      *reinterpret_cast<Pack<T, VE>*>(static_cast<T*>(a.out) + token * a.width + c) = p;
    }
  }
  if (!a.dots) return;  // the whole grid alike
#pragma unroll
  for (int j = 0; j < S; ++j) {
    if (j >= a.per_token) break;
    dot[j] = warp_sum(dot[j]);
    if (NW > 1 && (threadIdx.x & 31) == 0) part[threadIdx.x >> 5][j] = dot[j];
  }
  if (NW > 1) __syncthreads();
#pragma unroll
  for (int j = 0; j < S; ++j) {
    if (j < a.per_token && t == 0) {
      float d = dot[j];
      if (NW > 1) {
#pragma unroll
        for (int w = 1; w < NW; ++w) d += part[w][j];
      }
      a.dots[slot0 + j] = d;
    }
  }
}

template <typename T, int NW, int VE>
int launch_join_s(const JoinArgs& a, cudaStream_t st) {
  const unsigned blocks = (unsigned)ceil_div(a.tokens, NW == 1 ? 8 : 1);
  constexpr int threads = NW == 1 ? 256 : NW * 32;
  if (a.per_token <= 2)
    join_kernel<T, NW, 2, VE><<<blocks, threads, 0, st>>>(a);
  else if (a.per_token <= 4)
    join_kernel<T, NW, 4, VE><<<blocks, threads, 0, st>>>(a);
  else if (a.per_token <= 8)
    join_kernel<T, NW, 8, VE><<<blocks, threads, 0, st>>>(a);
  else
    join_kernel<T, NW, 32, VE><<<blocks, threads, 0, st>>>(a);
  return check_launch("expert_linear join");
}

template <typename T>
int launch_join(const JoinArgs& a, cudaStream_t st) {
  if (a.tokens == 0) return FSC_OK;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vec = a.width % 4 == 0 && al(a.x) && al(a.out) && al(a.slot_out) && al(a.z);
  // A block a token where its threads have columns to take.  Forward with 4096 rows of 16 inputs, 4 slots, block and warp a
  // token, us: 128 bf16 columns 25 / 17, 256 28 / 20, 512 33 / 27, 1024 50 / 46, 2048 87 / 90; fp32 256 34 / 27,
  // 1024 63 / 60.
  const bool block = a.width >= 512;
  if constexpr (sizeof(T) == 2) {  // two slots: eight columns a thread, for as much in flight as with four slots
    if (vec && a.width % 8 == 0 && a.per_token <= 2) return block ? launch_join_s<T, 4, 8>(a, st) : launch_join_s<T, 1, 8>(a, st);
  }
  if (vec) return block ? launch_join_s<T, 8, 4>(a, st) : launch_join_s<T, 1, 4>(a, st);
  return block ? launch_join_s<T, 8, 1>(a, st) : launch_join_s<T, 1, 1>(a, st);
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
// PAIR: clusters of two blocks.  row_tiles: tiles of rows (or of outputs and parts), times those of features.
template <typename T, int PA, int PB, int NT, bool A_MN, bool DW, bool PROMOTE, bool PAIR, typename OUT>
int launch_blocks(const CUtensorMap& ma, const CUtensorMap& mb, ProductArgs a, int64_t row_tiles, cudaStream_t st) {
  a.tiles_m = (int)ceil_div(a.M, PAIR ? 2 * BM : BM);
  const int64_t tiles = row_tiles * a.tiles_m;
  FSC_REQUIRE(tiles < (1ll << 31) - 1024, "expert_linear: too many tiles");
  constexpr int smem = Shape<PA, PB, NT, PAIR>::SMEM;
  auto k = product_kernel<T, PA, PB, NT, A_MN, DW, PROMOTE, PAIR, OUT>;
  if (!allow_shared(k, smem)) return check_launch("expert_linear");
  const int64_t units = std::min<int64_t>(tiles, sm_count() / (PAIR ? 2 : 1));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(units * (PAIR ? 2 : 1)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute pair;
  pair.id = cudaLaunchAttributeClusterDimension;
  pair.val.clusterDim.x = 2, pair.val.clusterDim.y = 1, pair.val.clusterDim.z = 1;
  cfg.attrs = &pair;
  cfg.numAttrs = PAIR ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, k, ma, mb, a) != cudaSuccess) return check_launch("expert_linear product");
  return check_launch("expert_linear product");
}

template <typename T, int PA, int PB, int NT, bool A_MN, bool DW, bool PROMOTE, typename OUT>
int launch_product(const CUtensorMap& ma, const CUtensorMap& mb, const ProductArgs& a, int64_t row_tiles, cudaStream_t st) {
  // 32-bit operands keep single blocks: three planes of a pair's tile leave two stages, as they do now
  if constexpr (PA < 3) {
    if (a.M > BM) return launch_blocks<T, PA, PB, NT, A_MN, DW, PROMOTE, true, OUT>(ma, mb, a, row_tiles, st);
  }
  return launch_blocks<T, PA, PB, NT, A_MN, DW, PROMOTE, false, OUT>(ma, mb, a, row_tiles, st);
}

// Rows in the plan's order (times the slots' weights, if given) as an operand of P planes in the arena.
template <typename T, typename E, int P>
int sorted_operand(const Sizes& z, const ProductArgs& a, const void* in, int by_slot, int64_t cols, const float* weights,
                   Arena& arena, Operand<E>* o, cudaStream_t st) {
  const int64_t slots = z.tokens * z.per_token;
  const int64_t rows = slots * z.comps + 16 * std::min<int64_t>(z.experts, slots);
  *o = Operand<E>{nullptr, 1, rows, (int)cols, Of<T>::pitch(cols), P};
  E* buf = arena.take<E>(P * rows * o->pitch);
  o->p = buf;
  if (arena.measuring) return FSC_OK;
  FSC_REQUIRE(arena.ok(), "expert_linear: workspace too small");
  SortArgs g{in, buf, weights, a.offsets, a.order, a.experts, a.per_token, a.comps, by_slot, (int)cols, o->pitch, rows};
  const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(rows, 8), 148 * 8);
  if (cols % (16 / sizeof(T)) == 0)
    sort_kernel<T, E, P, true><<<blocks, 256, 0, st>>>(g);
  else
    sort_kernel<T, E, P, false><<<blocks, 256, 0, st>>>(g);
  return check_launch("expert_linear sort");
}

// Parts into which an expert's rows are cut for its weight gradient: enough tiles for every SM, and 1024
// rows or more in a part.  At least 256 / 1024 / 4096 rows, us: 32768 bf16 rows, 8 experts 256 x 256: 42 / 39 / 51;
// 65536 fp32 rows, 2 of 8 experts 64 x 64: 145 / 135 / 177; 16384 fp32 rows, 4 experts 128 x 128: 30 / 41 / 89.
int weight_splits(const Sizes& z) {
  const int64_t tiles = z.experts * ceil_div(z.inputs, BM) * ceil_div(z.outputs, 256);
  const int64_t most = std::max<int64_t>(1, z.tokens * z.per_token * z.comps / z.experts / 1024);
  return (int)std::max<int64_t>(1, std::min<int64_t>({ceil_div(148, tiles), most, 64}));
}

// One product of sorted rows `b` with the weights `w` into slot rows of type OUT.
template <typename T, bool TRANS, bool PROMOTE, typename OUT>
int rows_product(const Sizes& z, ProductArgs a, const Operand<typename Of<T>::E>& w, const Operand<typename Of<T>::E>& b,
                 int features, int contraction, void* out, cudaStream_t st) {
  using E = typename Of<T>::E;
  constexpr int P = Of<T>::P;
  constexpr int NT = P == 3 ? 128 : 256;
  CUtensorMap ma, mb;
  FSC_TRY(tile_map(&ma, w, TRANS ? 64 : BM, true));
  FSC_TRY(tile_map(&mb, b, 64, false));
  a.M = features, a.Kd = contraction, a.out = out;
  const int64_t slots = z.tokens * z.per_token;
  const int64_t tiles = ceil_div(slots * z.comps, NT) + std::min<int64_t>(z.experts, slots);
  return launch_product<E, P, P, NT, TRANS, false, PROMOTE, OUT>(ma, mb, a, tiles, st);
}

// The gradient in the weights from the sorted rows of x (times their weights) and of g.
template <typename T, typename E, int PA, int PB>
int weight_product(const Sizes& z, ProductArgs a, const Operand<E>& x, const Operand<E>& g, void* grad_w, Arena& arena,
                   cudaStream_t st) {
  constexpr int NT = PA == 3 ? 128 : 256;
  const int splits = weight_splits(z);
  const int64_t n = z.experts * z.outputs * z.inputs;
  float* part = splits > 1 ? arena.take<float>(splits * n) : nullptr;
  if (arena.measuring) return FSC_OK;
  FSC_REQUIRE(arena.ok(), "expert_linear_backward: workspace too small");
  CUtensorMap ma, mb;
  FSC_TRY(tile_map(&ma, x, 64, false));
  FSC_TRY(tile_map(&mb, g, 64, false));
  a.M = (int)z.inputs, a.N = (int)z.outputs;
  a.tiles_n = (int)ceil_div(z.outputs, NT), a.splits = splits;
  const int64_t tiles = z.experts * a.tiles_n * splits;
  if (splits == 1) {
    a.out = grad_w;
    return launch_product<E, PA, PB, NT, true, true, true, T>(ma, mb, a, tiles, st);
  }
  a.out = part;
  FSC_TRY((launch_product<E, PA, PB, NT, true, true, true, float>(ma, mb, a, tiles, st)));
  split_sum_kernel<T><<<(unsigned)std::min<int64_t>(ceil_div(n, 256), 148 * 8), 256, 0, st>>>(part, splits, n,
                                                                                              static_cast<T*>(grad_w));
  return check_launch("expert_linear weight gradient");
}

template <typename T, typename OUT>
int forward(const Sizes& z, ProductArgs a, const void* x, const void* w, const int32_t* indices, const float* weights,
            int x_by_slot, void* out, Arena& arena, cudaStream_t st) {
  const int64_t slots = z.tokens * z.per_token;
  Operand<typename Of<T>::E> ow, ox;
  a.x_by_slot = x_by_slot;
  FSC_TRY(weights_operand(static_cast<const T*>(w), z.experts, z.outputs, z.inputs, arena, &ow, st));
  FSC_TRY((sorted_operand<T, typename Of<T>::E, Of<T>::P>(z, a, x, x_by_slot, z.inputs, nullptr, arena, &ox, st)));
  constexpr bool PROMOTE = std::is_same<OUT, float>::value;
  if (weights == nullptr || z.per_token == 1) {  // a row of the output for each product: written directly
    if (arena.measuring) return FSC_OK;
    a.row_weight = weights;
    zero_slots_kernel<OUT><<<(unsigned)std::min<int64_t>(slots, 148 * 8), 256, 0, st>>>(
        indices, a.experts, slots, z.comps * z.outputs, static_cast<OUT*>(out));
    FSC_TRY(check_launch("expert_linear"));
    return rows_product<T, false, PROMOTE, OUT>(z, a, ow, ox, z.outputs, z.inputs, out, st);
  }
  float* buf = arena.take<float>(slots * z.comps * z.outputs);
  if (arena.measuring) return FSC_OK;
  FSC_REQUIRE(arena.ok(), "expert_linear: workspace too small");
  FSC_TRY((rows_product<T, false, PROMOTE, float>(z, a, ow, ox, z.outputs, z.inputs, buf, st)));
  JoinArgs j{};
  j.z = buf, j.indices = indices, j.weights = weights, j.out = out;
  j.tokens = z.tokens, j.per_token = a.per_token, j.experts = a.experts, j.width = z.comps * z.outputs;
  return launch_join<OUT>(j, st);
}

size_t joint_bytes(int dtype, const Sizes& z) {
  JointCall c{};
  c.experts = z.experts, c.inputs = z.inputs, c.outputs = z.outputs;
  size_t n = 0;
  joint_product(dtype, false, c, nullptr, &n, nullptr);
  return n;
}

template <typename T>
int backward(const Sizes& z, ProductArgs a, const void* grad_out, const void* x, const void* w, const int32_t* indices,
             const float* weights, int x_by_slot, int rows_wanted, void* grad_x, void* grad_w, float* grad_weights,
             const JointCall* joint, Arena& arena, cudaStream_t st) {
  using E = typename Of<T>::E;
  constexpr int P = Of<T>::P;
  constexpr int dtype = P == 3 ? FSC_F32 : std::is_same<T, __half>::value ? FSC_F16 : FSC_BF16;
  const int64_t slots = z.tokens * z.per_token;
  Operand<E> og, ow;
  if (joint && rows_wanted) {
    const size_t bytes = joint_bytes(dtype, z);
    char* buf = arena.take<char>(bytes);
    if (!arena.measuring) {
      FSC_REQUIRE(arena.ok(), "expert_linear_backward: workspace too small");
      JointCall c = *joint;
      c.workspace_bytes = bytes;
      FSC_TRY(joint_product(dtype, true, c, buf, nullptr, st));
    }
    rows_wanted = 0;
  }
  const bool scaled = P == 1 && weights != nullptr;  // 16-bit rows times their weights: two planes
  if (rows_wanted || (grad_w && !(scaled && std::is_same<T, __half>::value)))
    FSC_TRY((sorted_operand<T, E, P>(z, a, grad_out, weights == nullptr, z.outputs, nullptr, arena, &og, st)));
  if (rows_wanted) {
    FSC_TRY(weights_operand(static_cast<const T*>(w), z.experts, z.outputs, z.inputs, arena, &ow, st));
    float* buf = arena.take<float>(slots * z.comps * z.inputs);
    if (!arena.measuring) {
      FSC_REQUIRE(arena.ok(), "expert_linear_backward: workspace too small");
      if (P == 3 || grad_weights) {
        FSC_TRY((rows_product<T, true, true, float>(z, a, ow, og, z.inputs, z.outputs, buf, st)));
      } else if constexpr (P == 1) {
        FSC_TRY((rows_product<T, true, false, float>(z, a, ow, og, z.inputs, z.outputs, buf, st)));
      }
      JoinArgs j{};
      j.z = buf, j.indices = indices, j.weights = weights;
      j.tokens = z.tokens, j.per_token = a.per_token, j.experts = a.experts, j.width = z.comps * z.inputs;
      j.x = grad_weights ? x : nullptr, j.x_by_slot = x_by_slot, j.dots = grad_weights;
      (x_by_slot ? j.slot_out : j.out) = grad_x;
      FSC_TRY(launch_join<T>(j, st));
    }
  }
  if (grad_w == nullptr) return FSC_OK;
  if constexpr (P == 1) {
    // A row times its weight is not rounded to the rows' type: it is two bfloat16 (2^-16 of it, and nothing of it beyond
    // the range, as in fp16), and so is a row of g in fp16, exactly.  The gradient then has one rounding, its own, for
    // twice (fp16: three times) the products: 8192 bf16 rows, 2 of 8 experts 1024 x 2048, 123 us instead of 76 us.
    using B = __nv_bfloat16;
    if (scaled) {
      Operand<B> ox;
      FSC_TRY((sorted_operand<T, B, 2>(z, a, x, x_by_slot, z.inputs, weights, arena, &ox, st)));
      if constexpr (std::is_same<T, B>::value) {
        return weight_product<T, B, 2, 1>(z, a, ox, og, grad_w, arena, st);
      } else {
        Operand<B> ob;
        FSC_TRY((sorted_operand<T, B, 2>(z, a, grad_out, 0, z.outputs, nullptr, arena, &ob, st)));
        return weight_product<T, B, 2, 2>(z, a, ox, ob, grad_w, arena, st);
      }
    }
  }
  Operand<E> ox;
  FSC_TRY((sorted_operand<T, E, P>(z, a, x, x_by_slot, z.inputs, weights, arena, &ox, st)));
  return weight_product<T, E, P, P>(z, a, ox, og, grad_w, arena, st);
}

ProductArgs common(const Sizes& z, const int32_t* offsets, const int32_t* order, int32_t* status) {
  ProductArgs a{};
  a.offsets = offsets, a.order = order, a.status = status;
  a.experts = (int)z.experts, a.per_token = (int)z.per_token, a.comps = (int)z.comps;
  return a;
}

// Bytes of a forward product; q8: from e4m3.
size_t forward_bytes(int dtype, const Sizes& z, int x_by_slot, bool weighted, bool q8) {
  Arena arena(nullptr, 0);
  const float* w = weighted ? reinterpret_cast<const float*>(16) : nullptr;
  by_type(q8 ? FSC_F32 : dtype, [&](auto t) {
    using T = decltype(t);
    ProductArgs a{};
    return q8 ? forward<e4m3, float>(z, a, nullptr, nullptr, nullptr, w, x_by_slot, nullptr, arena, nullptr)
              : forward<T, T>(z, a, nullptr, nullptr, nullptr, w, x_by_slot, nullptr, arena, nullptr);
  });
  return arena.off;
}

}  // namespace
}  // namespace fsc

using namespace fsc;

extern "C" {

size_t fsc_expert_linear_workspace_bytes(int dtype, int64_t tokens, int64_t per_token, int64_t comps, int64_t experts,
                                         int64_t inputs, int64_t outputs, int x_by_slot, int weighted, int joint) {
  const Sizes z{tokens, per_token, comps, experts, inputs, outputs};
  if ((!float_type(dtype) && dtype != FSC_E4M3) || check_sizes(z) != FSC_OK || tokens == 0) return 0;
  if (joint && weighted && !x_by_slot && dtype != FSC_E4M3 &&
      joint_fits(dtype, tokens, per_token, comps, experts, outputs, inputs))
    return joint_bytes(dtype, z);
  return forward_bytes(dtype, z, x_by_slot != 0, weighted != 0, dtype == FSC_E4M3);
}

int fsc_expert_linear(int dtype, const void* x, const void* w, const int32_t* indices, const float* weights,
                      const int32_t* offsets, const int32_t* order, const int32_t* joint_offsets,
                      const int32_t* joint_order, int32_t* status, void* out, int64_t tokens, int64_t per_token,
                      int64_t comps, int64_t experts, int64_t inputs, int64_t outputs, int x_by_slot, void* workspace,
                      size_t workspace_bytes, void* stream) {
  const Sizes z{tokens, per_token, comps, experts, inputs, outputs};
  FSC_REQUIRE(float_type(dtype), "expert_linear: dtype must be f32, bf16 or f16");
  FSC_TRY(check_sizes(z));
  if (tokens == 0) return FSC_OK;
  FSC_REQUIRE(x && w && indices && offsets && order && status && out, "expert_linear: null pointer");
  FSC_REQUIRE(al16({x, w, out, workspace}), "expert_linear: x, w, out and workspace must start on 16 bytes");
  const bool joint = joint_offsets && joint_order;
  const size_t need = fsc_expert_linear_workspace_bytes(dtype, tokens, per_token, comps, experts, inputs, outputs, x_by_slot,
                                                        weights != nullptr, joint);
  FSC_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "expert_linear: workspace too small");
  if (joint && weights && !x_by_slot && joint_fits(dtype, tokens, per_token, comps, experts, outputs, inputs)) {
    const JointCall c{x,     nullptr, w,      weights,   joint_offsets, joint_order, status, out,
                      nullptr, tokens,  per_token, comps,     experts,       inputs,      outputs, workspace_bytes};
    return joint_product(dtype, false, c, workspace, nullptr, as_stream(stream));
  }
  Arena arena(workspace ? workspace : reinterpret_cast<void*>(16), workspace_bytes);
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    return forward<T, T>(z, common(z, offsets, order, status), x, w, indices, weights, x_by_slot != 0, out, arena,
                         as_stream(stream));
  });
}

int fsc_expert_linear_q8(int out_dtype, const void* x, const float* x_scale, const void* w, const float* w_scale,
                         const int32_t* indices, const float* weights, const int32_t* offsets, const int32_t* order,
                         int32_t* status, void* out, int64_t tokens, int64_t per_token, int64_t comps,
                         int64_t experts, int64_t inputs, int64_t outputs, int x_by_slot, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const Sizes z{tokens, per_token, comps, experts, inputs, outputs};
  FSC_REQUIRE(float_type(out_dtype), "expert_linear_q8: out_dtype must be f32, bf16 or f16");
  FSC_REQUIRE(comps == 1, "expert_linear_q8: rows have one component");
  FSC_TRY(check_sizes(z));
  if (tokens == 0) return FSC_OK;
  FSC_REQUIRE(x && x_scale && w && w_scale && indices && offsets && order && status && out,
              "expert_linear_q8: null pointer");
  FSC_REQUIRE(al16({x, w, out, workspace}), "expert_linear_q8: x, w, out and workspace must start on 16 bytes");
  const size_t need = forward_bytes(FSC_E4M3, z, x_by_slot != 0, weights != nullptr, true);
  FSC_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "expert_linear_q8: workspace too small");
  Arena arena(workspace ? workspace : reinterpret_cast<void*>(16), workspace_bytes);
  ProductArgs a = common(z, offsets, order, status);
  a.x_scale = x_scale, a.w_scale = w_scale;
  return by_type(out_dtype, [&](auto t) {
    return forward<e4m3, decltype(t)>(z, a, x, w, indices, weights, x_by_slot != 0, out, arena, as_stream(stream));
  });
}

size_t fsc_expert_linear_backward_workspace_bytes(int dtype, int64_t tokens, int64_t per_token, int64_t comps,
                                                  int64_t experts, int64_t inputs, int64_t outputs, int x_by_slot,
                                                  int weighted, int rows_gradient, int weight_gradient, int joint) {
  const Sizes z{tokens, per_token, comps, experts, inputs, outputs};
  if (!float_type(dtype) || check_sizes(z) != FSC_OK || tokens == 0) return 0;
  Arena arena(nullptr, 0);
  const JointCall c{};
  const bool fits = joint && weighted && !x_by_slot && joint_fits(dtype, tokens, per_token, comps, experts, inputs, outputs);
  by_type(dtype, [&](auto t) {
    return backward<decltype(t)>(z, ProductArgs{}, nullptr, nullptr, nullptr, nullptr,
                                 weighted ? reinterpret_cast<const float*>(16) : nullptr, x_by_slot != 0, rows_gradient != 0,
                                 nullptr, weight_gradient ? reinterpret_cast<void*>(16) : nullptr, nullptr, fits ? &c : nullptr,
                                 arena, nullptr);
  });
  return arena.off;
}

int fsc_expert_linear_backward(int dtype, const void* grad_out, const void* x, const void* w, const int32_t* indices,
                               const float* weights, const int32_t* offsets, const int32_t* order,
                               const int32_t* joint_offsets, const int32_t* joint_order, int32_t* status, void* grad_x,
                               void* grad_w, float* grad_weights, int64_t tokens, int64_t per_token, int64_t comps,
                                int64_t experts, int64_t inputs, int64_t outputs, int x_by_slot,
                               void* workspace, size_t workspace_bytes, void* stream) {
  const Sizes z{tokens, per_token, comps, experts, inputs, outputs};
  FSC_REQUIRE(float_type(dtype), "expert_linear_backward: dtype must be f32, bf16 or f16");
  FSC_TRY(check_sizes(z));
  cudaStream_t st = as_stream(stream);
  if (tokens == 0) {
    const size_t n = (size_t)(experts * outputs) * (size_t)inputs * (dtype == FSC_F32 ? 4 : 2);
    if (grad_w && cudaMemsetAsync(grad_w, 0, n, st) != cudaSuccess) return check_launch("expert_linear_backward");
    return FSC_OK;
  }
  FSC_REQUIRE(grad_out && x && w && indices && offsets && order && status, "expert_linear_backward: null pointer");
  FSC_REQUIRE(!grad_weights || weights, "expert_linear_backward: grad_weights needs weights");
  FSC_REQUIRE(al16({grad_out, x, w, grad_x, grad_w, workspace}),
              "expert_linear_backward: tensors and workspace must start on 16 bytes");
  const int rows = grad_x != nullptr || grad_weights != nullptr;
  const bool joint = joint_offsets && joint_order;
  const bool fits = joint && weights && !x_by_slot && joint_fits(dtype, tokens, per_token, comps, experts, inputs, outputs);
  const JointCall c{grad_out, grad_weights ? x : nullptr, w,         weights, joint_offsets, joint_order, status, grad_x,
                    grad_weights, tokens,             per_token, comps,   experts,       inputs,      outputs, 0};
  const size_t need = fsc_expert_linear_backward_workspace_bytes(dtype, tokens, per_token, comps, experts, inputs, outputs,
                                                                 x_by_slot, weights != nullptr, rows, grad_w != nullptr, joint);
  FSC_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "expert_linear_backward: workspace too small");
  Arena arena(workspace ? workspace : reinterpret_cast<void*>(16), workspace_bytes);
  return by_type(dtype, [&](auto t) {
    return backward<decltype(t)>(z, common(z, offsets, order, status), grad_out, x, w, indices, weights, x_by_slot != 0,
                                 rows, grad_x, grad_w, grad_weights, fits ? &c : nullptr, arena, st);
  });
}

}  // extern "C"
