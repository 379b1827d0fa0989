// Mixture of experts: y_n = sum_j gate_nj (gelu(x_n W1_e + b1_e) W2_e + b2_e), e = idx_nj,
// and its gradients, on tcgen05.  (No counterpart in the reference; the dense MLP it
// replaces is dtrain/nn.py:90-101.)
//
// Rows are the (token, slot) pairs that have an expert, sorted by expert; each expert's
// rows start at a multiple of 64 and are padded with zero rows to the next one, so that
// a k-block of 64 rows never mixes two experts' rows in the weight gradients.
//
//   moe_hist / moe_offsets / moe_place   the plan: a stable counting sort of the slots
//   moe_gather        xp[r] = x[token of r]
//   grouped GEMMs     pre = xp W1 + b1, act = gelu(pre) ; yp = act W2 + b2
//   moe_combine       y[n] = sum_j gate_nj yp[row of (n, j)]
//   moe_grad_rows     u[r] = gate dy[token of r],  dgate = dy . yp[r]
//   grouped GEMMs     dpre = (u W2^T) gelu'(pre) ; dxp = dpre W1^T
//   grouped GEMMs     dW2_e = act_e^T u_e ; dW1_e = xp_e^T dpre_e   (over the expert's rows)
//   moe_col_sums      db2_e, db1_e
//
// The number of rows of each expert stays on the device: grids are sized by the most
// tiles that the slots can fill, and the kernels read the real counts from the plan.
// Every sum has a fixed order (no float atomics).
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros_like.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "gemm_tile.cuh"

namespace dtb {

constexpr int kMoeMaxExperts = 512;
constexpr int kMoeMaxK = 32;
constexpr int kRowPad = 64;

// The plan (int32), sized by the most rows and tiles that P slots and E experts can have.
struct MoePlan {
  int4* tile;  // row tiles of 128 in expert order: {expert, first row, end of the expert's rows, 0}
  int* ntile;  // [1], padded to 4
  int* off;    // [E + 1] first row of each expert, a multiple of 64
  int* count;  // [E] rows of each expert, without the padding
  int* inv;    // [P] row of a slot, -1: none
  int* src;    // [R] slot of a row, -1: padding
  int* hist;   // [blocks, E] scratch
};
static long moe_max_rows(long P, long E) {
  return (P + (kRowPad - 1) * std::min(P, E) + kRowPad - 1) / kRowPad * kRowPad;
}
static long moe_max_tiles(long P, long E) { return P / kBM + std::min(P, E); }
constexpr int kPlanThreads = 256;
constexpr int kPlanChunk = 2048;  // slots a block sorts: 8 warps x 256
static long plan_blocks(long P) { return std::max<long>(1, (P + kPlanChunk - 1) / kPlanChunk); }
static long plan_ints(long P, long E) {
  return 4 * moe_max_tiles(P, E) + 4 + (E + 1) + E + P + moe_max_rows(P, E) + plan_blocks(P) * E;
}
static MoePlan plan_views(int* p, long P, long E) {
  MoePlan v;
  v.tile = reinterpret_cast<int4*>(p);
  v.ntile = p + 4 * moe_max_tiles(P, E);
  v.off = v.ntile + 4;
  v.count = v.off + E + 1;
  v.inv = v.count + E;
  v.src = v.inv + P;
  v.hist = v.src + moe_max_rows(P, E);
  return v;
}

template <typename I>
__device__ __forceinline__ int slot_expert(const I* idx, long s, int E) {
  const I v = idx[s];
  return (v >= 0 && v < (I)E) ? (int)v : -1;
}

template <typename I>
__global__ void __launch_bounds__(kPlanThreads) moe_hist_kernel(const I* __restrict__ idx, long P, int E, MoePlan pl) {
  extern __shared__ int s_h[];
  for (int i = threadIdx.x; i < E; i += blockDim.x) s_h[i] = 0;
  __syncthreads();
  const long lo = (long)blockIdx.x * kPlanChunk, hi = min(P, lo + kPlanChunk);
  for (long s = lo + threadIdx.x; s < hi; s += blockDim.x) {
    const int e = slot_expert(idx, s, E);
    if (e >= 0) atomicAdd(&s_h[e], 1);
    else if (idx[s] >= (I)E) set_status(kStatusBadArgument);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < E; i += blockDim.x) pl.hist[(long)blockIdx.x * E + i] = s_h[i];
}

// One block of 512 threads (one per expert): totals, offsets, and each block's start in its experts' rows.
__global__ void __launch_bounds__(kMoeMaxExperts) moe_offsets_kernel(int nb, int E, MoePlan pl) {
  __shared__ int s_a[kMoeMaxExperts], s_b[kMoeMaxExperts];
  const int e = threadIdx.x;
  int total = 0;
  if (e < E)
    for (int b = 0; b < nb; ++b) total += pl.hist[(long)b * E + e];
  const int padded = (total + kRowPad - 1) / kRowPad * kRowPad;
  s_a[e] = e < E ? padded : 0;
  s_b[e] = e < E ? (padded + kBM - 1) / kBM : 0;
  __syncthreads();
  for (int o = 1; o < kMoeMaxExperts; o <<= 1) {
    const int a = e >= o ? s_a[e - o] : 0, b = e >= o ? s_b[e - o] : 0;
    __syncthreads();
    s_a[e] += a;
    s_b[e] += b;
    __syncthreads();
  }
  if (e < E) {
    const int start = s_a[e] - padded;
    pl.count[e] = total;
    pl.off[e + 1] = s_a[e];
    const int tiles = (padded + kBM - 1) / kBM;
    for (int t = 0; t < tiles; ++t) pl.tile[s_b[e] - tiles + t] = make_int4(e, start + t * kBM, s_a[e], 0);
    if (e == E - 1) pl.ntile[0] = s_b[e];
    int at = start;
    for (int b = 0; b < nb; ++b) {
      const long h = (long)b * E + e;
      const int c = pl.hist[h];
      pl.hist[h] = at;
      at += c;
    }
    for (int r = start + total; r < start + padded; ++r) pl.src[r] = -1;
  }
  if (e == 0) pl.off[0] = 0;
}

// Each warp places 256 slots in a row: first it counts its experts, then (after the
// warps before it are known) it gives the slots their rows in order.
template <typename I>
__global__ void __launch_bounds__(kPlanThreads) moe_place_kernel(const I* __restrict__ idx, long P, int E, MoePlan pl) {
  extern __shared__ int s_w[];  // [8][E]
  constexpr int W = kPlanThreads / 32, PER = kPlanChunk / W;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < W * E; i += blockDim.x) s_w[i] = 0;
  __syncthreads();
  int* mine = s_w + warp * E;
  const long base = (long)blockIdx.x * kPlanChunk + warp * PER;
  for (int i = lane; i < PER; i += 32) {
    const int e = base + i < P ? slot_expert(idx, base + i, E) : -1;
    if (e >= 0) atomicAdd(&mine[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    int at = pl.hist[(long)blockIdx.x * E + e];
    for (int w = 0; w < W; ++w) {
      const int c = s_w[w * E + e];
      s_w[w * E + e] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int i = lane; i < PER; i += 32) {
    const long s = base + i;
    const int e = s < P ? slot_expert(idx, s, E) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1u));
    int row = -1;
    if (e >= 0) row = mine[e] + rank;
    __syncwarp();
    if (e >= 0 && rank == 0) mine[e] += __popc(same);
    __syncwarp();
    if (s < P) {
      pl.inv[s] = row;
      if (row >= 0) pl.src[row] = (int)s;
    }
  }
}

// ---------------------------------------------------------------- rows in and out
__device__ __forceinline__ void unpack8(const uint4& u, float* v) {
  const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ float load_gate(const float* g, long i) { return g[i]; }
__device__ __forceinline__ float load_gate(const bf16* g, long i) { return bf2f(g[i]); }
__device__ __forceinline__ void store_gate(float* g, long i, float v) { g[i] = v; }
__device__ __forceinline__ void store_gate(bf16* g, long i, float v) { g[i] = f2bf(v); }

// One warp per row; padding rows become zeros.
__global__ void __launch_bounds__(256)
    moe_gather_kernel(const bf16* __restrict__ x, bf16* __restrict__ xp, MoePlan pl, int E, int C, int k) {
  const int lane = threadIdx.x & 31;
  const int rows = pl.off[E];
  for (int r = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; r < rows; r += (gridDim.x * blockDim.x) >> 5) {
    const int s = pl.src[r];
    uint4* dst = reinterpret_cast<uint4*>(xp + (long)r * C);
    if (s < 0) {
      for (int c = lane; c < C / 8; c += 32) dst[c] = make_uint4(0, 0, 0, 0);
    } else {
      const uint4* p = reinterpret_cast<const uint4*>(x + (long)(s / k) * C);
      for (int c = lane; c < C / 8; c += 32) dst[c] = p[c];
    }
  }
}

// One warp per token: y = sum over its slots of gate * yp[row] (gates null: of yp[row]).
template <typename G>
__global__ void __launch_bounds__(256)
    moe_combine_kernel(const bf16* __restrict__ yp, const G* __restrict__ gates, bf16* __restrict__ y, MoePlan pl,
                       int n, int C, int k) {
  const int lane = threadIdx.x & 31;
  for (int t = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; t < n; t += (gridDim.x * blockDim.x) >> 5) {
    for (int c = lane; c < C / 8; c += 32) {
      float acc[8] = {};
      for (int j = 0; j < k; ++j) {
        const long s = (long)t * k + j;
        const int r = pl.inv[s];
        if (r < 0) continue;
        const float g = gates ? load_gate(gates, s) : 1.f;
        float v[8];
        unpack8(*reinterpret_cast<const uint4*>(yp + (long)r * C + c * 8), v);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = fmaf(g, v[i], acc[i]);
      }
      *reinterpret_cast<uint4*>(y + (long)t * C + c * 8) = pack8(acc);
    }
  }
}

// One warp per row: u = gate * dy[token], d(gate) = dy[token] . yp[row].  u is rounded to
// bf16: it is the tensor cores' operand in three products.
template <typename G>
__global__ void __launch_bounds__(256)
    moe_grad_rows_kernel(const bf16* __restrict__ dy, const bf16* __restrict__ yp, const G* __restrict__ gates,
                         bf16* __restrict__ u, G* __restrict__ dgates, MoePlan pl, int E, int C, int k) {
  const int lane = threadIdx.x & 31;
  const int rows = pl.off[E];
  for (int r = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; r < rows; r += (gridDim.x * blockDim.x) >> 5) {
    const int s = pl.src[r];
    uint4* dst = reinterpret_cast<uint4*>(u + (long)r * C);
    if (s < 0) {
      for (int c = lane; c < C / 8; c += 32) dst[c] = make_uint4(0, 0, 0, 0);
      continue;
    }
    const float g = load_gate(gates, s);
    const uint4* d = reinterpret_cast<const uint4*>(dy + (long)(s / k) * C);
    const uint4* o = reinterpret_cast<const uint4*>(yp + (long)r * C);
    float dot = 0.f;
    for (int c = lane; c < C / 8; c += 32) {
      float a[8], b[8];
      unpack8(d[c], a);
      unpack8(o[c], b);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dot = fmaf(a[i], b[i], dot);
        a[i] *= g;
      }
      dst[c] = pack8(a);
    }
#pragma unroll
    for (int o2 = 16; o2; o2 >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o2);
    if (lane == 0) store_gate(dgates, s, dot);
  }
}

// out[e, c] = sum over the expert's rows of g[r, c]: one block per expert and 64 columns,
// 32 row lanes x 8 column vectors, joined in a fixed order.
template <typename O>
__global__ void __launch_bounds__(256)
    moe_col_sums_kernel(const bf16* __restrict__ g, O* __restrict__ out, MoePlan pl, int N) {
  __shared__ float s_sum[32][65];
  const int e = blockIdx.y, c0 = blockIdx.x * 64;
  const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
  const int lo = pl.off[e], hi = lo + pl.count[e];
  const int c = c0 + tx * 8;
  float acc[8] = {};
  if (c < N)
    for (int r = lo + ty; r < hi; r += 32) {
      float v[8];
      unpack8(*reinterpret_cast<const uint4*>(g + (long)r * N + c), v);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += v[i];
    }
#pragma unroll
  for (int i = 0; i < 8; ++i) s_sum[ty][tx * 8 + i] = acc[i];
  __syncthreads();
  if (threadIdx.x < 64 && c0 + threadIdx.x < N) {
    float s = 0.f;
    for (int r = 0; r < 32; ++r) s += s_sum[r][threadIdx.x];
    store_gate(out, (long)e * N + c0 + threadIdx.x, s);
  }
}

// ---------------------------------------------------------------- grouped GEMM
enum MoeMode : int {
  MOE_FWD = 0,  // out rows = A rows . W_e        (W_e stored [K, N])
  MOE_DX = 1,   // out rows = A rows . W_e^T      (W_e stored [N, K])
  MOE_DW = 2,   // out_e = A_e^T . B_e over the expert's rows
};
enum MoeEpi : int {
  MOE_PLAIN = 0,  // out = acc [+ bias_e], bf16
  MOE_GELU = 1,   // out = gelu(acc [+ bias_e]); aux = acc [+ bias_e] where asked for
  MOE_DGELU = 2,  // out = acc * gelu'(aux)
  MOE_F32 = 3,    // out = acc, fp32
};
struct MoeGemmArgs {
  const int4* tile;  // row tiles, and their number
  const int* ntile;
  const int* off;    // [E + 1] first row of each expert
  int E, M, N, K;   // M, K: the sizes that are not rows
  int epi;
  const bf16* bias;    // [E, N] or null
  const bf16* aux_in;  // [R, N]
  int save_aux;
};

// Where unit u of the grid lies: expert, first row and column of the tile, end of its rows, first row
// (MOE_DW) and number of the k-blocks.
struct MoeUnit {
  int e, m0, n0, row_end, r0, kb;
};
template <int MODE, int BM, int BN>
__device__ __forceinline__ MoeUnit moe_unit(const MoeGemmArgs& a, int u, int mt, int nt) {
  MoeUnit q;
  int mi, ni;
  if (MODE == MOE_DW) {
    q.e = u / (mt * nt);
    tile_coords(u - q.e * mt * nt, mt, nt, mi, ni);
    q.m0 = mi * BM;
    q.row_end = a.M;
    q.r0 = __ldg(a.off + q.e);
    q.kb = (__ldg(a.off + q.e + 1) - q.r0) / kBK;
  } else {
    tile_coords(u, mt, nt, mi, ni);
    const int4 t = __ldg(a.tile + mi);
    q.e = t.x;
    q.m0 = t.y;
    q.row_end = t.z;
    q.r0 = 0;
    q.kb = (a.K + kBK - 1) / kBK;
  }
  q.n0 = ni * BN;
  return q;
}

// One 32x32 chunk: this lane's row of 32 accumulators -> slab -> TMA store.
__device__ __forceinline__ void moe_epi_chunk(const MoeGemmArgs& a, const CUtensorMap* tmOut, const CUtensorMap* tmAux,
                                              uint8_t* slab, int lane, int row0, int col, int e, bool dw, float* v) {
  switch (a.epi) {
    case MOE_PLAIN:
    case MOE_GELU: {
      if (a.bias) {
        float b[32];
        load_row32(a.bias + (long)e * a.N, col, a.N, b);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] += b[j];
      }
      if (a.epi == MOE_GELU) {
        if (a.save_aux) slab_put_bf16(slab + 2048, lane, v);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = gelu_fast(v[j]);
      }
      slab_put_bf16(slab, lane, v);
      break;
    }
    case MOE_DGELU: {
      float h[32];
      load_row32(a.aux_in + (long)(row0 + lane) * a.N, col, a.N, h);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= gelu_grad_fast(h[j]);
      slab_put_bf16(slab, lane, v);
      break;
    }
    case MOE_F32: {
      slab_put_f32(slab, lane, v);
      break;
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    if (dw) {
      tma_store_3d(tmOut, slab, col, row0, e);
    } else {
      if (a.epi == MOE_GELU && a.save_aux) tma_store_2d(tmAux, slab + 2048, col, row0);
      tma_store_2d(tmOut, slab, col, row0);
    }
    bulk_commit();
  }
}

template <int BN>
struct MoeCfg {
  static constexpr int A_BYTES = kBM * kBK * 2;
  static constexpr int B_BYTES = BN * kBK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = (BN == 256) ? 4 : 5;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int EPI_BYTES = kEpiWarps * kEpiSlab;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_BYTES + 1024 /*align*/ + 256 /*barriers*/;
};

template <int BN, int MODE>
__global__ void __maxnreg__(DTB_CORESIDENT_MAXNREG)
    moe_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ CUtensorMap tmAux,
                    MoeGemmArgs args) {
  using Cfg = MoeCfg<BN>;
  constexpr bool A_MN = MODE == MOE_DW, B_MN = MODE != MOE_DX;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi_smem = smem + Cfg::STAGES * Cfg::STAGE_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(epi_smem + Cfg::EPI_BYTES);
  uint64_t* empty_bar = full_bar + Cfg::STAGES;
  uint64_t* tfull_bar = empty_bar + Cfg::STAGES;  // [2]
  uint64_t* tempty_bar = tfull_bar + 2;           // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull_bar[b], 1);
      mbar_init(&tempty_bar[b], kEpiWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int nt = (args.N + BN - 1) / BN;
  const int mt = MODE == MOE_DW ? (args.M + kBM - 1) / kBM : __ldg(args.ntile);
  const int units = MODE == MOE_DW ? args.E * mt * nt : mt * nt;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------------ TMA producer
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        const MoeUnit q = moe_unit<MODE, kBM, BN>(args, u, mt, nt);
        for (int kb = 0; kb < q.kb; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag)) { ok = false; break; }
          uint8_t* sA = smem + stage * Cfg::STAGE_BYTES;
          uint8_t* sB = sA + Cfg::A_BYTES;
          mbar_arrive_expect_tx(&full_bar[stage], Cfg::STAGE_BYTES);
          if (MODE == MOE_DW) {
            const int r0 = q.r0 + kb * kBK;
#pragma unroll
            for (int c = 0; c < kBM / 64; ++c) tma_load_2d(&tmA, sA + c * 8192, &full_bar[stage], q.m0 + c * 64, r0);
#pragma unroll
            for (int c = 0; c < BN / 64; ++c) tma_load_2d(&tmB, sB + c * 8192, &full_bar[stage], q.n0 + c * 64, r0);
          } else {
            const int k0 = kb * kBK;
            tma_load_2d(&tmA, sA, &full_bar[stage], k0, q.m0);
            if (MODE == MOE_DX) {
              tma_load_3d(&tmB, sB, &full_bar[stage], k0, q.n0, q.e);
            } else {
#pragma unroll
              for (int c = 0; c < BN / 64; ++c)
                tma_load_3d(&tmB, sB + c * 8192, &full_bar[stage], q.n0 + c * 64, k0, q.e);
            }
          }
          if (++stage == Cfg::STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ------------------------------------------------------------ MMA issuer
      constexpr uint32_t idesc = make_idesc_bf16(kBM, BN, A_MN, B_MN);
      int stage = 0;
      uint32_t phase = 0;
      int ab = 0;
      uint32_t aphase = 0;
      bool ok = true;
      for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
        const MoeUnit q = moe_unit<MODE, kBM, BN>(args, u, mt, nt);
        if (q.kb == 0) continue;  // an expert without rows: the epilogue writes zeros
        if (!mbar_wait(&tempty_bar[ab], aphase ^ 1, abort_flag)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(ab * BN);
        for (int kb = 0; kb < q.kb; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint32_t aBase = smem_u32(smem + stage * Cfg::STAGE_BYTES);
          const uint32_t bBase = aBase + Cfg::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk) {
            const uint64_t ad = A_MN ? make_sw128_desc(aBase + kk * 2048, 8192, 1024)
                                     : make_sw128_desc(aBase + kk * 32, 16, 1024);
            const uint64_t bd = B_MN ? make_sw128_desc(bBase + kk * 2048, 8192, 1024)
                                     : make_sw128_desc(bBase + kk * 32, 16, 1024);
            tc_mma_f16(d_tmem, ad, bd, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
          }
          tc_commit(&empty_bar[stage]);
          if (++stage == Cfg::STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tc_commit(&tfull_bar[ab]);
        if (++ab == 2) { ab = 0; aphase ^= 1; }
      }
    }
  } else {
    // -------------------------------------------------------------- epilogue
    const int ew = warp - 2;
    const int q4 = warp & 3;
    const int half = ew >> 2;
    uint8_t* slab = epi_smem + ew * kEpiSlab;
    // one bf16 output a chunk: the slab's halves alternate; two outputs or fp32 fill it
    const bool dbl = args.epi == MOE_PLAIN || args.epi == MOE_DGELU || (args.epi == MOE_GELU && !args.save_aux);
    uint32_t ck = 0;
    int ab = 0;
    uint32_t aphase = 0;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      const MoeUnit q = moe_unit<MODE, kBM, BN>(args, u, mt, nt);
      if (q.kb > 0) {
        if (!mbar_wait(&tfull_bar[ab], aphase, abort_flag)) break;
        tc_fence_after();
      }
      const int row0 = q.m0 + q4 * 32;
      const uint32_t tbase = tmem_base + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(ab * BN);
      const int c_begin = half * (BN / 2), c_end = c_begin + BN / 2;
      if (row0 < q.row_end) {  // rows of the next expert (or past the matrix) are not this tile's
#pragma unroll 1
        for (int c = c_begin; c < c_end; c += 32) {
          if (q.n0 + c >= args.N) break;
          float v[32];
          if (q.kb > 0) {
            tmem_ld32(tbase + c, v);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0.f;
          }
          epi_slab_acquire(lane, dbl);
          moe_epi_chunk(args, &tmOut, &tmAux, slab + (dbl ? (ck & 1) * 2048 : 0), lane, row0, q.n0 + c, q.e,
                        MODE == MOE_DW, v);
          ++ck;
        }
      }
      if (q.kb > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty_bar[ab]);
        if (++ab == 2) { ab = 0; aphase ^= 1; }
      }
    }
    if (lane == 0) bulk_wait0();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

// ------------------------------------------------------------------ host
// 3-D bf16 operand map over [depth, rows, cols], 128B swizzle: a box never leaves its expert's matrix
// (rows and columns past its end read as zeros).
static CUtensorMap make_map3(const void* base, long depth, long rows, long cols, int box_cols, int box_rows) {
  CUtensorMap m;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)depth};
  cuuint64_t strides[2] = {(cuuint64_t)cols * 2, (cuuint64_t)cols * rows * 2};
  cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = get_encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box,
                               estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code ", (int)r);
  return m;
}

template <int BN, int MODE>
static void launch_moe(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& to, const CUtensorMap& tx,
                       const MoeGemmArgs& a, long units, cudaStream_t st) {
  static bool attr_set = false;
  auto kern = moe_gemm_kernel<BN, MODE>;
  if (!attr_set) {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, MoeCfg<BN>::SMEM_BYTES);
    attr_set = true;
  }
  const int grid = (int)std::min<long>(units, num_sms());
  kern<<<grid, kThreads, MoeCfg<BN>::SMEM_BYTES, st>>>(ta, tb, to, tx, a);
  count_launch();
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

struct MoeSizes {
  long n, k, P, E, R;  // tokens, slots a token, slots, experts, most padded rows
};

// rows [R, N] = rows [R, K] . W_e (MOE_FWD, w [E, K, N]) or . W_e^T (MOE_DX, w [E, N, K])
static void moe_rows_gemm(int mode, const bf16* a, const bf16* w, bf16* out, int N, int K, int epi, const bf16* bias,
                          bf16* aux, const MoePlan& pl, const MoeSizes& z, cudaStream_t st) {
  MoeGemmArgs g{};
  g.off = pl.off;
  g.tile = pl.tile;
  g.ntile = pl.ntile;
  g.E = (int)z.E;
  g.N = N;
  g.K = K;
  g.M = 1;
  g.epi = epi;
  g.bias = bias;
  g.aux_in = aux;
  g.save_aux = epi == MOE_GELU && aux != nullptr;
  const int bn = N <= 128 ? 128 : 256;
  const CUtensorMap ta = make_map(a, z.R, K, K, 64, kBM);
  const CUtensorMap tb = mode == MOE_FWD ? make_map3(w, z.E, K, N, 64, 64) : make_map3(w, z.E, N, K, 64, bn);
  const CUtensorMap to = make_store_map(out, false, z.R, N, N);
  const CUtensorMap tx = g.save_aux ? make_store_map(aux, false, z.R, N, N) : to;
  const long units = moe_max_tiles(z.P, z.E) * ((N + bn - 1) / bn);
  if (mode == MOE_FWD) {
    if (bn == 256) launch_moe<256, MOE_FWD>(ta, tb, to, tx, g, units, st);
    else launch_moe<128, MOE_FWD>(ta, tb, to, tx, g, units, st);
  } else {
    if (bn == 256) launch_moe<256, MOE_DX>(ta, tb, to, tx, g, units, st);
    else launch_moe<128, MOE_DX>(ta, tb, to, tx, g, units, st);
  }
}

// out_e [M, N] (fp32 or bf16) = a_e^T . b_e over the expert's rows
static void moe_weight_gemm(const bf16* a, const bf16* b, at::Tensor& out, int M, int N, const MoePlan& pl,
                            const MoeSizes& z, cudaStream_t st) {
  MoeGemmArgs g{};
  g.off = pl.off;
  g.E = (int)z.E;
  g.M = M;
  g.N = N;
  const bool f32 = out.scalar_type() == at::kFloat;
  g.epi = f32 ? MOE_F32 : MOE_PLAIN;
  const int bn = N <= 128 ? 128 : 256;
  const CUtensorMap ta = make_map(a, z.R, M, M, 64, 64);
  const CUtensorMap tb = make_map(b, z.R, N, N, 64, 64);
  const CUtensorMap to = make_store_map(out.data_ptr(), f32, M, N, N, z.E);
  const long units = z.E * ((M + kBM - 1) / kBM) * ((N + bn - 1) / bn);
  if (bn == 256) launch_moe<256, MOE_DW>(ta, tb, to, to, g, units, st);
  else launch_moe<128, MOE_DW>(ta, tb, to, to, g, units, st);
}

static int warp_grid(long rows) { return (int)std::max<long>(1, std::min<long>((rows + 7) / 8, 148L * 8)); }

static void moe_build_plan(const at::Tensor& idx, const MoePlan& pl, const MoeSizes& z, cudaStream_t st) {
  const int nb = (int)plan_blocks(z.P), E = (int)z.E;
  if (idx.scalar_type() == at::kInt) {
    moe_hist_kernel<int><<<nb, kPlanThreads, E * 4, st>>>(idx.data_ptr<int>(), z.P, E, pl);
    moe_offsets_kernel<<<1, kMoeMaxExperts, 0, st>>>(nb, E, pl);
    moe_place_kernel<int><<<nb, kPlanThreads, 8 * E * 4, st>>>(idx.data_ptr<int>(), z.P, E, pl);
  } else {
    const long* p = reinterpret_cast<const long*>(idx.data_ptr<int64_t>());
    moe_hist_kernel<long><<<nb, kPlanThreads, E * 4, st>>>(p, z.P, E, pl);
    moe_offsets_kernel<<<1, kMoeMaxExperts, 0, st>>>(nb, E, pl);
    moe_place_kernel<long><<<nb, kPlanThreads, 8 * E * 4, st>>>(p, z.P, E, pl);
  }
  count_launch(3);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

static const bf16* bptr(const at::Tensor& t) { return reinterpret_cast<const bf16*>(t.data_ptr()); }
static bf16* bptr_mut(const at::Tensor& t) { return reinterpret_cast<bf16*>(t.data_ptr()); }
static const bf16* bptr_opt(const std::optional<at::Tensor>& t) {
  return t && t->defined() ? bptr(*t) : nullptr;
}

static void check_bf16(const at::Tensor& t, const at::Tensor& x, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.get_device() == x.get_device(), "experts: ", what, " must be on x's CUDA device");
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 && t.is_contiguous(), "experts: ", what, " must be contiguous bf16");
  TORCH_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0, "experts: ", what, " must be 16-byte aligned");
}

static MoeSizes check_experts(const at::Tensor& x, const at::Tensor& w1, const std::optional<at::Tensor>& b1,
                              const at::Tensor& w2, const std::optional<at::Tensor>& b2,
                              const at::Tensor& gates) {
  check_bf16(x, x, "x");
  check_bf16(w1, x, "w1");
  check_bf16(w2, x, "w2");
  TORCH_CHECK(x.dim() == 2 && w1.dim() == 3 && w2.dim() == 3, "experts: x [n, c], w1 [e, c, h], w2 [e, h, co] expected");
  const long E = w1.size(0), C = w1.size(1), H = w1.size(2), Co = w2.size(2);
  TORCH_CHECK(x.size(1) == C && w2.size(0) == E && w2.size(1) == H, "experts: x ", x.sizes(), ", w1 ", w1.sizes(),
              " and w2 ", w2.sizes(), " do not fit");
  TORCH_CHECK(E >= 1 && E <= kMoeMaxExperts, "experts: 1 to ", kMoeMaxExperts, " experts, got ", E);
  TORCH_CHECK(C % 8 == 0 && H % 8 == 0 && Co % 8 == 0 && C > 0 && H > 0 && Co > 0,
              "experts: widths must be multiples of 8, got ", C, ", ", H, ", ", Co);
  if (b1 && b1->defined()) {
    check_bf16(*b1, x, "b1");
    TORCH_CHECK(b1->dim() == 2 && b1->size(0) == E && b1->size(1) == H, "experts: b1 must be [experts, h]");
  }
  if (b2 && b2->defined()) {
    check_bf16(*b2, x, "b2");
    TORCH_CHECK(b2->dim() == 2 && b2->size(0) == E && b2->size(1) == Co, "experts: b2 must be [experts, co]");
  }
  TORCH_CHECK(gates.is_cuda() && gates.get_device() == x.get_device() && gates.dim() == 2 &&
                  gates.size(0) == x.size(0) && gates.is_contiguous() &&
                  (gates.scalar_type() == at::kFloat || gates.scalar_type() == at::kBFloat16),
              "experts: gates must be contiguous fp32 or bf16 [n, k] on x's device");
  MoeSizes z;
  z.n = x.size(0);
  z.k = gates.size(1);
  z.E = E;
  TORCH_CHECK(z.k >= 1 && z.k <= kMoeMaxK, "experts: 1 to ", kMoeMaxK, " slots a token, got ", z.k);
  z.P = z.n * z.k;
  z.R = moe_max_rows(z.P, E);
  TORCH_CHECK(z.R < (1L << 31) - 256, "experts: too many rows");
  return z;
}

// Forward.  Returns [y] or, with `save`, [y, plan, xp, pre, act, yp] for experts_bwd.
std::vector<at::Tensor> experts_fwd(at::Tensor x, at::Tensor w1, std::optional<at::Tensor> b1,
                                       at::Tensor w2, std::optional<at::Tensor> b2, at::Tensor idx,
                                       at::Tensor gates, bool save) {
  const MoeSizes z = check_experts(x, w1, b1, w2, b2, gates);
  TORCH_CHECK(idx.is_cuda() && idx.get_device() == x.get_device() && idx.sizes() == gates.sizes() &&
                  idx.is_contiguous() && (idx.scalar_type() == at::kInt || idx.scalar_type() == at::kLong),
              "experts: idx must be contiguous int32 or int64, of the gates' shape");
  c10::cuda::CUDAGuard guard(x.device());
  bind_device_context(x.get_device());
  const long C = w1.size(1), H = w1.size(2), Co = w2.size(2);
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  auto y = at::empty({z.n, Co}, x.options());
  if (z.n == 0) {
    if (!save) return {y};
    auto none = at::empty({0}, x.options());
    return {y, none, none, none, none, none};
  }
  auto plan = at::empty({plan_ints(z.P, z.E)}, x.options().dtype(at::kInt));
  const MoePlan pl = plan_views(plan.data_ptr<int>(), z.P, z.E);
  moe_build_plan(idx, pl, z, st);
  auto xp = at::empty({z.R, C}, x.options());
  moe_gather_kernel<<<warp_grid(z.R), 256, 0, st>>>(bptr(x), bptr_mut(xp), pl, (int)z.E, (int)C, (int)z.k);
  count_launch();
  auto act = at::empty({z.R, H}, x.options());
  at::Tensor pre;
  if (save) pre = at::empty({z.R, H}, x.options());
  auto yp = at::empty({z.R, Co}, x.options());
  moe_rows_gemm(MOE_FWD, bptr(xp), bptr(w1), bptr_mut(act), (int)H, (int)C, MOE_GELU, bptr_opt(b1),
                save ? bptr_mut(pre) : nullptr, pl, z, st);
  moe_rows_gemm(MOE_FWD, bptr(act), bptr(w2), bptr_mut(yp), (int)Co, (int)H, MOE_PLAIN, bptr_opt(b2), nullptr, pl, z,
                st);
  if (gates.scalar_type() == at::kFloat)
    moe_combine_kernel<float><<<warp_grid(z.n), 256, 0, st>>>(bptr(yp), gates.data_ptr<float>(), bptr_mut(y), pl,
                                                             (int)z.n, (int)Co, (int)z.k);
  else
    moe_combine_kernel<bf16><<<warp_grid(z.n), 256, 0, st>>>(bptr(yp), bptr(gates), bptr_mut(y), pl, (int)z.n, (int)Co,
                                                            (int)z.k);
  count_launch();
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (!save) return {y};
  return {y, plan, xp, pre, act, yp};
}

// Backward: returns [dx, dgates]; the weights' and biases' gradients are written to dw1, db1, dw2, db2
// (all bf16 or all fp32; db1 / db2 only where the layer has the bias).
std::vector<at::Tensor> experts_bwd(at::Tensor dy, at::Tensor x, at::Tensor w1, at::Tensor w2,
                                       at::Tensor gates, std::vector<at::Tensor> saved, at::Tensor dw1,
                                       std::optional<at::Tensor> db1, at::Tensor dw2,
                                       std::optional<at::Tensor> db2) {
  const MoeSizes z = check_experts(x, w1, std::nullopt, w2, std::nullopt, gates);
  const long C = w1.size(1), H = w1.size(2), Co = w2.size(2);
  check_bf16(dy, x, "dy");
  TORCH_CHECK(dy.dim() == 2 && dy.size(0) == z.n && dy.size(1) == Co, "experts_bwd: dy must be [n, co]");
  TORCH_CHECK(saved.size() == 5, "experts_bwd: the forward's plan, xp, pre, act and yp expected");
  const auto wt = dw1.scalar_type();
  TORCH_CHECK(wt == at::kFloat || wt == at::kBFloat16, "experts_bwd: fp32 or bf16 weight gradients");
  const auto check_grad = [&](const at::Tensor& t, at::IntArrayRef sizes, const char* what) {
    TORCH_CHECK(t.is_cuda() && t.get_device() == x.get_device() && t.scalar_type() == wt && t.sizes() == sizes &&
                    t.is_contiguous() && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0,
                "experts_bwd: ", what, " must be a contiguous, 16-byte aligned ", wt, " tensor of its weight's shape");
  };
  check_grad(dw1, w1.sizes(), "dw1");
  check_grad(dw2, w2.sizes(), "dw2");
  if (db1 && db1->defined()) check_grad(*db1, {z.E, H}, "db1");
  if (db2 && db2->defined()) check_grad(*db2, {z.E, Co}, "db2");
  c10::cuda::CUDAGuard guard(x.device());
  bind_device_context(x.get_device());
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  auto dx = at::empty({z.n, C}, x.options());
  auto dgates = at::zeros_like(gates);
  if (z.n == 0) {
    dw1.zero_();
    dw2.zero_();
    if (db1 && db1->defined()) db1->zero_();
    if (db2 && db2->defined()) db2->zero_();
    return {dx, dgates};
  }
  const at::Tensor &plan = saved[0], &xp = saved[1], &pre = saved[2], &act = saved[3], &yp = saved[4];
  TORCH_CHECK(plan.scalar_type() == at::kInt && plan.numel() == plan_ints(z.P, z.E) && xp.size(0) == z.R &&
                  xp.size(1) == C && pre.size(0) == z.R && pre.size(1) == H && act.sizes() == pre.sizes() &&
                  yp.size(0) == z.R && yp.size(1) == Co,
              "experts_bwd: saved tensors of another forward");
  const MoePlan pl = plan_views(plan.data_ptr<int>(), z.P, z.E);
  const bool gf = gates.scalar_type() == at::kFloat;
  auto u = at::empty({z.R, Co}, x.options());
  if (gf)
    moe_grad_rows_kernel<float><<<warp_grid(z.R), 256, 0, st>>>(bptr(dy), bptr(yp), gates.data_ptr<float>(),
                                                               bptr_mut(u), dgates.data_ptr<float>(), pl, (int)z.E,
                                                               (int)Co, (int)z.k);
  else
    moe_grad_rows_kernel<bf16><<<warp_grid(z.R), 256, 0, st>>>(bptr(dy), bptr(yp), bptr(gates), bptr_mut(u),
                                                              bptr_mut(dgates), pl, (int)z.E, (int)Co, (int)z.k);
  count_launch();
  const auto col_sums = [&](const at::Tensor& g, const std::optional<at::Tensor>& out, long N) {
    if (!out || !out->defined()) return;
    const dim3 grid((unsigned)((N + 63) / 64), (unsigned)z.E);
    if (wt == at::kFloat) moe_col_sums_kernel<float><<<grid, 256, 0, st>>>(bptr(g), out->data_ptr<float>(), pl, (int)N);
    else moe_col_sums_kernel<bf16><<<grid, 256, 0, st>>>(bptr(g), bptr_mut(*out), pl, (int)N);
    count_launch();
  };
  auto dpre = at::empty({z.R, H}, x.options());
  moe_rows_gemm(MOE_DX, bptr(u), bptr(w2), bptr_mut(dpre), (int)H, (int)Co, MOE_DGELU, nullptr, bptr_mut(pre), pl, z,
                st);
  moe_weight_gemm(bptr(act), bptr(u), dw2, (int)H, (int)Co, pl, z, st);
  col_sums(u, db2, Co);
  auto dxp = at::empty({z.R, C}, x.options());
  moe_rows_gemm(MOE_DX, bptr(dpre), bptr(w1), bptr_mut(dxp), (int)C, (int)H, MOE_PLAIN, nullptr, nullptr, pl, z, st);
  moe_weight_gemm(bptr(xp), bptr(dpre), dw1, (int)C, (int)H, pl, z, st);
  col_sums(dpre, db1, H);
  moe_combine_kernel<float><<<warp_grid(z.n), 256, 0, st>>>(bptr(dxp), nullptr, bptr_mut(dx), pl, (int)z.n, (int)C,
                                                           (int)z.k);
  count_launch();
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {dx, dgates};
}

DTB_DEFINE_STATUS_READER(status_moe)

}  // namespace dtb
