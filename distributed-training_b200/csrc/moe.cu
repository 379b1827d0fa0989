// Mixture of experts: y_n = sum_j gate_nj (gelu(x_n W1_e + b1_e) W2_e + b2_e), e = idx_nj,
// and its gradients, on tcgen05.  (No counterpart in the reference; the dense MLP it
// replaces is dtrain/nn.py:90-101.)
//
// Rows are the (token, slot) pairs that have an expert, sorted by expert; each expert's
// rows start at a multiple of 64 and are padded with zero rows to the next one, so that
// a k-block of 64 rows never mixes two experts' rows in the weight gradients.
//
//   moe_plan          a stable counting sort of the slots by expert (three kernels for many slots)
//   moe_gather        xp[r] = x[token of r]
//   grouped GEMMs     pre = xp W1 + b1, act = gate gelu(pre) ; yp = act W2 + gate b2
//   moe_combine       y[n] = sum_j yp[row of (n, j)]
//   moe_dy_rows       dyp[r] = dy[token of r], sums of gate dyp for db2, dyp . b2
//   grouped GEMMs     t = dyp W2^T: dpre = gate t gelu'(pre), and t . gelu(pre) (d(gate), with dyp . b2) ; dxp = dpre W1^T
//   grouped GEMMs     dW2_e = act_e^T dyp_e ; dW1_e = xp_e^T dpre_e   (over the expert's rows)
//   moe_join_sums     db2_e, db1_e from sums over blocks of rows
//   moe_combine       dx[n] = sum_j dxp[row of (n, j)], d(gate)
//
// The gates are applied in the epilogues, so the backward reads neither the rows' outputs nor a scaled copy of dy.
//
// Sums are fp32 (in the products, over a token's slots, over rows).  What is rounded to bf16 on the way, and why;
// errors in the 2-norm relative to 64 bits, 512 tokens, 4 experts of 768 x 1536, 2 slots a token, where the results'
// own rounding to bf16 is 0.0017:
//   act, dpre    operands of a tensor core product.  With them every result but d(gate) is off by 0.0023.
//   pre          saved for the backward's gelu and its slope: d(gate) 0.0027 (exact pre: 0.0017), dx and dW1 0.0024.
//                In fp32 it would be twice the bytes of the largest tensor that the backward reads.
//   yp, dxp      each slot's part of y and dx: 0.0029 and 0.0030 (in fp32 0.0023 and 0.0024, as the forms for few rows
//                have it, whose parts stay in L2).  Stored in fp32 the pass forward and backward took 1155 us
//                for 1088 (16384 tokens, 16 experts 768 x 1536) and 1859 for 1777 (8192, 32 of 2048 x 2048).
// db1 sums dpre as rounded, as its product does.  tanh.approx is off by 2^-11 at most, a quarter of the
// largest bf16 rounding.
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

// Programmatic dependent launch: a kernel that is launched this way may start while the one before it runs.
// pdl_wait returns once that one is complete and its writes are visible; pdl_launch lets the next one start.
// Kernels here call pdl_launch after pdl_wait, so what a kernel's own predecessor waited for is complete too.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

constexpr int kMoeMaxExperts = 512;
constexpr int kMoeMaxK = 32;
constexpr int kRowPad = 64;

// The plan (int32), sized by the most rows and tiles that P slots and E experts can have.
struct MoePlan {
  int4* tile;   // row tiles of 128 in expert order: {expert, first row, end of the expert's rows, 0}
  int4* tile2;  // the same of 256 rows
  int4* tile3;  // and of 64, with the end of the expert's rows that are not padding; their number is off[E] / 64
  int* ntile;   // [2] the numbers of the first two, padded to 4
  int* off;    // [E + 1] first row of each expert, a multiple of 64
  int* order;  // [E] the experts by falling number of rows
  int* inv;    // [P] row of a slot, -1: none
  int* src;    // [R] slot of a row, -1: padding
  int* hist;   // [E, blocks] scratch: rows of each expert in a block of slots, then its first row there
};
static long moe_max_rows(long P, long E) {
  return (P + (kRowPad - 1) * std::min(P, E) + kRowPad - 1) / kRowPad * kRowPad;
}
static long moe_max_tiles(long P, long E) { return P / kBM + std::min(P, E); }
constexpr int kPlanThreads = 256;
constexpr int kPlanChunk = 1024;  // slots a block sorts: 8 warps x 128
static long plan_blocks(long P) { return std::max<long>(1, (P + kPlanChunk - 1) / kPlanChunk); }
static long plan_ints(long P, long E) {
  return 8 * moe_max_tiles(P, E) + moe_max_rows(P, E) / kRowPad * 4 + 4 + (E + 1) + E + P + moe_max_rows(P, E) + plan_blocks(P) * E;
}
static MoePlan plan_views(int* p, long P, long E) {
  MoePlan v;
  v.tile = reinterpret_cast<int4*>(p);
  v.tile2 = v.tile + moe_max_tiles(P, E);
  v.tile3 = v.tile2 + moe_max_tiles(P, E);
  v.ntile = reinterpret_cast<int*>(v.tile3 + moe_max_rows(P, E) / kRowPad);
  v.src = v.ntile + 4;
  v.off = v.src + moe_max_rows(P, E);
  v.order = v.off + E + 1;
  v.inv = v.order + E;
  v.hist = v.inv + P;
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
  pdl_launch();
  for (int i = threadIdx.x; i < E; i += blockDim.x) s_h[i] = 0;
  __syncthreads();
  const long lo = (long)blockIdx.x * kPlanChunk, hi = min(P, lo + kPlanChunk);
  for (long s = lo + threadIdx.x; s < hi; s += blockDim.x) {
    const int e = slot_expert(idx, s, E);
    if (e >= 0) atomicAdd(&s_h[e], 1);
    else if (idx[s] >= (I)E) set_status(kStatusBadArgument);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < E; i += blockDim.x) pl.hist[(long)i * gridDim.x + blockIdx.x] = s_h[i];
}

// Inclusive sums over the block's 512 threads of (a, b, c); every thread calls it.
__device__ __forceinline__ void plan_scan(int& a, int& b, int& c) {
  __shared__ int s_t[3][kMoeMaxExperts / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o),
              z = __shfl_up_sync(0xffffffffu, c, o);
    if (lane >= o) { a += x; b += y; c += z; }
  }
  if (lane == 31) { s_t[0][warp] = a; s_t[1][warp] = b; s_t[2][warp] = c; }
  __syncthreads();
  for (int w = 0; w < warp; ++w) { a += s_t[0][w]; b += s_t[1][w]; c += s_t[2][w]; }
}

// Thread e of 512: expert e's offsets and tiles from its number of rows; returns its first row.
__device__ __forceinline__ int plan_expert(const MoePlan& pl, int e, int E, int total) {
  const int padded = (total + kRowPad - 1) / kRowPad * kRowPad;
  const int t1 = (padded + kBM - 1) / kBM, t2 = (padded + 2 * kBM - 1) / (2 * kBM);
  int end = padded, n1 = t1, n2 = t2;
  __shared__ int s_total[kMoeMaxExperts];
  s_total[e] = total;
  plan_scan(end, n1, n2);  // (synchronises)
  const int start = end - padded;
  if (e < E) {
    int place = 0;
    for (int o = 0; o < E; ++o) place += s_total[o] > total || (s_total[o] == total && o < e);
    pl.order[place] = e;
    pl.off[e + 1] = end;
    if (e == 0) pl.off[0] = 0;
    for (int t = 0; t < t1; ++t) pl.tile[n1 - t1 + t] = make_int4(e, start + t * kBM, end, 0);
    for (int t = 0; t < t2; ++t) pl.tile2[n2 - t2 + t] = make_int4(e, start + t * 2 * kBM, end, 0);
    for (int r = start; r < end; r += kRowPad) pl.tile3[r / kRowPad] = make_int4(e, r, start + total, 0);
    if (e == E - 1) {
      pl.ntile[0] = n1;
      pl.ntile[1] = n2;
    }
    for (int r = start + total; r < end; ++r) pl.src[r] = -1;
  }
  return start;
}

// One block of 512 threads: totals (a warp per expert over the blocks' counts), offsets (a thread per expert), and
// each block's first row of its experts (a warp per expert again).
__global__ void __launch_bounds__(kMoeMaxExperts) moe_offsets_kernel(int nb, int E, MoePlan pl) {
  __shared__ int s_e[kMoeMaxExperts];
  pdl_wait();
  pdl_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = warp; e < E; e += kMoeMaxExperts / 32) {
    int t = 0;
    for (int b = lane; b < nb; b += 32) t += __ldcg(pl.hist + (long)e * nb + b);
    t = __reduce_add_sync(0xffffffffu, t);
    if (lane == 0) s_e[e] = t;
  }
  __syncthreads();
  const int mine = threadIdx.x < E ? s_e[threadIdx.x] : 0;
  const int start = plan_expert(pl, threadIdx.x, E, mine);
  s_e[threadIdx.x] = start;
  __syncthreads();
  for (int e = warp; e < E; e += kMoeMaxExperts / 32) {
    int at = s_e[e];
    for (int b0 = 0; b0 < nb; b0 += 32) {
      const long i = (long)e * nb + b0 + lane;
      const int c = b0 + lane < nb ? __ldcg(pl.hist + i) : 0;
      int sum = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
      if (b0 + lane < nb) pl.hist[i] = at + sum - c;
      at += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
}

// A warp gives the slots [base, base + count) their rows, in order; `next` holds its experts' next rows.
template <typename I>
__device__ __forceinline__ void place_slots(const I* idx, long base, int count, long P, int E, int* next,
                                            const MoePlan& pl) {
  const int lane = threadIdx.x & 31;
  for (int i = lane; i < count; i += 32) {
    const long s = base + i;
    const int e = s < P ? slot_expert(idx, s, E) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int rank = __popc(same & ((1u << lane) - 1u));
    int row = -1;
    if (e >= 0) row = next[e] + rank;
    __syncwarp();
    if (e >= 0 && rank == 0) next[e] += __popc(same);
    __syncwarp();
    if (s < P) {
      pl.inv[s] = row;
      if (row >= 0) pl.src[row] = (int)s;
    }
  }
}

// The whole plan in one block, for up to kPlanSmall slots: 16 warps count and place a sixteenth each.
// (2.6 us where the three kernels take 7.4, at 96 slots.)
constexpr int kPlanSmall = 4096;
template <typename I>
__global__ void __launch_bounds__(kMoeMaxExperts) moe_plan_kernel(const I* __restrict__ idx, int P, int E, MoePlan pl) {
  extern __shared__ int s_w[];  // [16][E]
  pdl_launch();
  constexpr int W = kMoeMaxExperts / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = ((P + W - 1) / W + 31) / 32 * 32;
  for (int i = threadIdx.x; i < W * E; i += blockDim.x) s_w[i] = 0;
  __syncthreads();
  for (int i = lane; i < per; i += 32) {
    const int s = warp * per + i;
    if (s < P) {
      const int e = slot_expert(idx, s, E);
      if (e >= 0) atomicAdd(&s_w[warp * E + e], 1);
      else if (idx[s] >= (I)E) set_status(kStatusBadArgument);
    }
  }
  __syncthreads();
  const int e = threadIdx.x;
  int total = 0;
  if (e < E)
    for (int w = 0; w < W; ++w) total += s_w[w * E + e];
  int at = plan_expert(pl, e, E, total);
  if (e < E)
    for (int w = 0; w < W; ++w) {
      const int c = s_w[w * E + e];
      s_w[w * E + e] = at;
      at += c;
    }
  __syncthreads();
  place_slots(idx, (long)warp * per, per, P, E, s_w + warp * E, pl);
}

// Each warp places 128 slots in a row: first it counts its experts, then (after the
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
  pdl_wait();
  pdl_launch();
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    int at = __ldcg(pl.hist + (long)e * gridDim.x + blockIdx.x);
    for (int w = 0; w < W; ++w) {
      const int c = s_w[w * E + e];
      s_w[w * E + e] = at;
      at += c;
    }
  }
  __syncthreads();
  place_slots(idx, base, PER, P, E, mine, pl);
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
  pdl_wait();
  pdl_launch();
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

// One warp per token: y = sum over its slots of rows[row].  The rows are read once, four slots' loads in
// flight a lane; bound by memory.  In the backward also the token's d(gate): the parts of its row's
// product that the dpre GEMM left, in order, and its product with the bias.
struct GateParts {
  const float* part;  // [parts, R], or null
  const float* bias;  // [bias_parts, R], or null
  int parts, bias_parts;
  long R;
};
template <typename G>
__global__ void __launch_bounds__(256)
    moe_combine_kernel(const bf16* __restrict__ rows, bf16* __restrict__ y, G* __restrict__ dgates, GateParts gp,
                       MoePlan pl, int n, int C, int k) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  for (int t = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; t < n; t += (gridDim.x * blockDim.x) >> 5) {
    int row = -1;
    if (lane < k) row = pl.inv[(long)t * k + lane];
    for (int c0 = 0; c0 < C / 8; c0 += 32) {
      const int c = c0 + lane;
      float acc[8] = {};
      for (int j = 0; j < k; j += 4) {
        uint4 u[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = __shfl_sync(0xffffffffu, row, (j + q) & 31);
          const bool there = j + q < k && r >= 0 && c < C / 8;
          u[q] = there ? __ldcs(reinterpret_cast<const uint4*>(rows + (long)r * C) + c) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[8];
          unpack8(u[q], v);
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i] += v[i];
        }
      }
      if (c < C / 8) *(reinterpret_cast<uint4*>(y + (long)t * C) + c) = pack8(acc);
    }
    if (gp.part != nullptr && lane < k) {
      float d = 0.f;
      if (row >= 0) {
#pragma unroll 8
        for (int p = 0; p < gp.parts; ++p) d += gp.part[(long)p * gp.R + row];
        if (gp.bias != nullptr)
          for (int p = 0; p < gp.bias_parts; ++p) d += gp.bias[(long)p * gp.R + row];
      }
      store_gate(dgates, (long)t * k + lane, d);
    }
  }
}

// A block of 64 rows (one expert's) and 256 columns per CTA, 8 rows a warp, 16 bytes a lane: dyp[r] = dy[token of r]
// (zeros: padding) and, where the layer has b2, the column sums of gate * dyp (db2's parts) and the columns' part of
// dyp . b2_e (for d(gate)).  Bound by the rows' way to DRAM; dy itself stays in L2.  Warps hide the loads' latency:
// whole rows of 768 (2048) columns a CTA, with 128 (166) registers a thread, took 61 (162) us for 65536 (32768) rows.
// (The grouped GEMMs could fetch the tokens' rows themselves, four a TMA gather, and no copy would be made.  The gather
// moves a row of 128 bytes in 24 cycles an SM: the first product of 65536 rows x 1536, K 768, took 418 us that way and
// takes 153 from a copy that costs 25.)
template <typename G>
__global__ void __launch_bounds__(256, 5)
    moe_dy_rows_kernel(const bf16* __restrict__ dy, const bf16* __restrict__ b2, const G* __restrict__ gates,
                       bf16* __restrict__ dyp, float* __restrict__ sums, float* __restrict__ dots, MoePlan pl, int E,
                       int C, int k, long R) {
  __shared__ float s_sum[8][256];
  pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int blocks = pl.off[E] / kRowPad;
  const int c0 = blockIdx.y * 256, c = c0 + lane * 8;
  const bool in = c < C;
  for (int b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int r0 = b * kRowPad + warp * 8;
    const int slot = lane < 8 ? pl.src[r0 + lane] : -1;
    const float gate = b2 && slot >= 0 ? load_gate(gates, slot) : 0.f;
    uint4 bv = make_uint4(0, 0, 0, 0);
    if (b2 && in) bv = *reinterpret_cast<const uint4*>(b2 + (long)pl.tile3[b].x * C + c);
    float dot = 0.f;  // lane i: row i's
    float acc[8] = {};
#pragma unroll
    for (int i0 = 0; i0 < 8; i0 += 4) {
      uint4 u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int s = __shfl_sync(0xffffffffu, slot, i0 + i);
        u[i] = s >= 0 && in ? __ldg(reinterpret_cast<const uint4*>(dy + (long)(s / k) * C + c)) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (in) *reinterpret_cast<uint4*>(dyp + (long)(r0 + i0 + i) * C + c) = u[i];
        if (b2) {
          const int s = __shfl_sync(0xffffffffu, slot, i0 + i);
          const float g = __shfl_sync(0xffffffffu, gate, i0 + i);
          float p = 0.f;
          if (s >= 0) {  // a padding row takes part in no sum (the bias need not be finite)
            float a[8], w[8];
            unpack8(u[i], a);
            unpack8(bv, w);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              p = fmaf(a[x], w[x], p);
              acc[x] = fmaf(g, a[x], acc[x]);
            }
          }
#pragma unroll
          for (int o2 = 16; o2; o2 >>= 1) p += __shfl_xor_sync(0xffffffffu, p, o2);
          if (lane == i0 + i) dot = p;
        }
      }
    }
    if (b2) {
#pragma unroll
      for (int x = 0; x < 8; x += 4)
        *reinterpret_cast<float4*>(&s_sum[warp][lane * 8 + x]) = make_float4(acc[x], acc[x + 1], acc[x + 2], acc[x + 3]);
      __syncthreads();
      if (c0 + (int)threadIdx.x < C) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) t += s_sum[w][threadIdx.x];
        sums[(long)b * C + c0 + threadIdx.x] = t;
      }
      __syncthreads();
      if (lane < 8) dots[(long)blockIdx.y * R + r0 + lane] = dot;
    }
  }
}

// out[e, c] = sum of the partial column sums of the expert's blocks of `rows` rows: one CTA per expert and
// 64 columns, 16 block lanes x 16 column vectors, joined in a fixed order.
// Grid z: the layer's first bias, then its second (where it has them).
template <typename O>
struct JoinArgs {
  const float* part;
  O* out;
  int N, rows;
};
template <typename O>
__global__ void __launch_bounds__(256) moe_join_sums_kernel(JoinArgs<O> first, JoinArgs<O> second, MoePlan pl) {
  __shared__ float s_sum[16][68];
  pdl_wait();
  pdl_launch();
  const JoinArgs<O> a = blockIdx.z == 0 ? first : second;
  const float* __restrict__ part = a.part;
  O* __restrict__ out = a.out;
  const int N = a.N, rows = a.rows;
  const int e = blockIdx.y, c0 = blockIdx.x * 64;
  if (c0 >= N) return;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int lo = pl.off[e] / rows, hi = pl.off[e + 1] / rows;
  const int c = c0 + tx * 4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < N)
#pragma unroll 4
    for (int r = lo + ty; r < hi; r += 16) {
      const float4 v = *reinterpret_cast<const float4*>(part + (long)r * N + c);
      acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
    }
  *reinterpret_cast<float4*>(&s_sum[ty][tx * 4]) = acc;
  __syncthreads();
  if (threadIdx.x < 64 && c0 + threadIdx.x < N) {
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) s += s_sum[r][threadIdx.x];
    store_gate(out, (long)e * N + c0 + threadIdx.x, s);
  }
}

// ---------------------------------------------------------------- a few slots (generation)
// For a token or a few the weights of the chosen experts are the whole work: they are
// streamed once by all SMs, without a plan, in two launches.
//   up    h[slot] = gelu(x W1_e + b1_e), fp32: a CTA per slot and 8 L columns, its threads in
//         512 / L rows of W1 by L 16-byte column vectors
//   down  y[n] = sum_j gate_j (h W2_e + b2_e): a cluster of 8 CTAs per token and 8 L columns;
//         each sums an eighth of the token's k H rows of W2, and the leader adds the eight
//         up in order through distributed shared memory
// `down` is launched while `up` runs (programmatic dependent launch) and asks for its weights
// in L2 before it waits for h, so both matrices stream at once.  L is 4, 8 or 16 by
// how many CTAs that makes.  The loads' latency is hidden by warps (512 threads, 64 registers;
// 256 threads took 26 us where this takes 19, 4 tokens of 16 experts 768 x 2048), and the last
// batch of a thread's loads is issued at once like the others.  One token there takes 9.6 us
// on the GPU for 12.6 MB (1.9 us at the copy rate): two launches, and in each the chain
// expert, weights, sum.
constexpr int kFewCluster = 8;
constexpr int kFewThreads = 512;

// acc (8 columns a thread) summed over the CTA's 512 / L row lanes: s_out[0 .. 8 L), valid after the
// __syncthreads that the caller does.
template <int L>
__device__ __forceinline__ void few_reduce(float* acc, float (*s_part)[8 * L], float* s_out) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int o = L; o < 32; o <<= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane < L) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s_part[warp][lane * 8 + i] = acc[i];
  }
  __syncthreads();
  if (threadIdx.x < 8 * L) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kFewThreads / 32; ++w) s += s_part[w][threadIdx.x];
    s_out[threadIdx.x] = s;
  }
}

__device__ __forceinline__ void few_fma(float* acc, const uint4& u, float x) {
  float w[8];
  unpack8(u, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = fmaf(x, w[i], acc[i]);
}

template <typename I, int L>
__global__ void __launch_bounds__(kFewThreads)
    moe_few_up_kernel(const bf16* __restrict__ x, const bf16* __restrict__ w1, const bf16* __restrict__ b1,
                      const I* __restrict__ idx, float* __restrict__ h, int E, int C, int H, int k) {
  __shared__ float s_part[kFewThreads / 32][8 * L];
  __shared__ float s_out[8 * L];
  extern __shared__ float s_x[];
  pdl_launch();
  const int slot = blockIdx.y;
  const int e = slot_expert(idx, slot, E);
  if (e < 0) {
    if (idx[slot] >= (I)E && threadIdx.x == 0) set_status(kStatusBadArgument);
    return;
  }
  const bf16* xr = x + (long)(slot / k) * C;
  for (int c = threadIdx.x; c < C / 8; c += kFewThreads) unpack8(*(reinterpret_cast<const uint4*>(xr) + c), s_x + c * 8);
  constexpr int R = kFewThreads / L;
  const int r = threadIdx.x / L, col = blockIdx.x * 8 * L + (threadIdx.x % L) * 8;
  __syncthreads();
  float acc[8] = {};
  if (col < H) {
    const uint4* w = reinterpret_cast<const uint4*>(w1 + (long)e * C * H + col);
    const long step = H / 8;
    constexpr int U = 6;  // loads in flight, the last batch's too
    for (int c = r; c < C; c += U * R) {
      uint4 u[U];
#pragma unroll
      for (int j = 0; j < U; ++j) u[j] = c + j * R < C ? __ldg(w + (c + j * R) * step) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < U; ++j)
        if (c + j * R < C) few_fma(acc, u[j], s_x[c + j * R]);
    }
  }
  few_reduce<L>(acc, s_part, s_out);
  const int oc = blockIdx.x * 8 * L + threadIdx.x;
  if (threadIdx.x < 8 * L && oc < H) {
    const float v = s_out[threadIdx.x] + (b1 ? bf2f(b1[(long)e * H + oc]) : 0.f);
    h[(long)slot * H + oc] = gelu_fast(v);
  }
}

template <typename I, typename G, int L>
__global__ void __cluster_dims__(kFewCluster, 1, 1) __launch_bounds__(kFewThreads)
    moe_few_down_kernel(const float* __restrict__ h, const bf16* __restrict__ w2, const bf16* __restrict__ b2,
                        const I* __restrict__ idx, const G* __restrict__ gates, bf16* __restrict__ y, int E, int H,
                        int Co, int k) {
  __shared__ float s_part[kFewThreads / 32][8 * L];
  __shared__ float s_out[8 * L];
  const int part = blockIdx.x;  // of the cluster
  const long n = blockIdx.z;
  constexpr int R = kFewThreads / L;
  const int r = threadIdx.x / L, col = blockIdx.y * 8 * L + (threadIdx.x % L) * 8;
  // each slot's rows [lo, hi) of this part
  const int lo = (int)((long)H * part / kFewCluster), hi = (int)((long)H * (part + 1) / kFewCluster);
  const long step = Co / 8;
  if (col < Co && (threadIdx.x % L) % 4 == 0)
    for (int j = 0; j < k; ++j) {
      const int e = slot_expert(idx, n * k + j, E);
      if (e < 0) continue;
      const uint4* w = reinterpret_cast<const uint4*>(w2 + (long)e * H * Co + col);
      for (int c = lo + r; c < hi; c += R) prefetch_l2(w + c * step);
    }
  pdl_wait();
  float acc[8] = {};
  for (int j = 0; j < k; ++j) {
    const int e = slot_expert(idx, n * k + j, E);
    if (e < 0 || col >= Co) continue;
    const float g = load_gate(gates, n * k + j);
    const uint4* w = reinterpret_cast<const uint4*>(w2 + (long)e * H * Co + col);
    const float* hr = h + (n * k + j) * H;
    constexpr int U = 4;
    for (int c = lo + r; c < hi; c += U * R) {
      uint4 u[U];
      float a[U];
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const bool there = c + q * R < hi;
        u[q] = there ? __ldg(w + (c + q * R) * step) : make_uint4(0, 0, 0, 0);
        a[q] = there ? __ldcg(hr + c + q * R) : 0.f;
      }
#pragma unroll
      for (int q = 0; q < U; ++q)
        if (c + q * R < hi) few_fma(acc, u[q], g * a[q]);
    }
  }
  few_reduce<L>(acc, s_part, s_out);
  cluster_sync_all();
  const int oc = blockIdx.y * 8 * L + threadIdx.x;
  if (part == 0 && threadIdx.x < 8 * L && oc < Co) {
    float v = 0.f;
#pragma unroll
    for (int p = 0; p < kFewCluster; ++p) {
      float t;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(t) : "r"(mapa_shared(&s_out[threadIdx.x], p)));
      v += t;
    }
    if (b2)
      for (int j = 0; j < k; ++j) {
        const int e = slot_expert(idx, n * k + j, E);
        if (e >= 0) v = fmaf(load_gate(gates, n * k + j), bf2f(b2[(long)e * Co + oc]), v);
      }
    y[n * Co + oc] = f2bf(v);
  }
  cluster_sync_all();  // the leader has read the others' sums
}

// ---------------------------------------------------------------- grouped GEMM
enum MoeMode : int {
  MOE_FWD = 0,  // out rows = A rows . W_e        (W_e stored [K, N])
  MOE_DX = 1,   // out rows = A rows . W_e^T      (W_e stored [N, K])
  MOE_DW = 2,   // out_e = A_e^T . B_e over the expert's rows
};
enum MoeEpi : int {
  MOE_PLAIN = 0,  // out = acc [+ gate * bias_e], bf16
  MOE_GELU = 1,   // out = gate * gelu(acc [+ bias_e]); aux = acc [+ bias_e] where asked for
  MOE_DGELU = 2,  // out = gate * acc * gelu'(aux), and the rows' products of acc with gelu(aux)
  MOE_F32 = 3,    // out = acc, fp32
};
struct MoeGemmArgs {
  const int4* tile;  // row tiles, and their number
  const int* ntile;
  const int* off;    // [E + 1] first row of each expert
  const int* order;  // [E] experts by falling number of rows
  int E, M, N, K;   // M, K: the sizes that are not rows
  int epi;
  const bf16* bias;    // [E, N] or null
  const bf16* aux_in;  // [R, N]
  int save_aux;
  float* sums;         // MOE_DGELU: [R / 32, N] column sums of each 32 rows of the output, or null
  float* dots;         // MOE_DGELU: [2 x tiles of N, R] each row's product of acc and gelu(aux), a half tile a part
  long R;
  const int* src;      // slot of a row, and the gates by slot (their type): the rows' gates, or null
  const void* gates;
  int gates_f32;
};

// Where unit u of the grid lies: expert, first row and column of the tile, end of its rows, first row
// (MOE_DW) and number of the k-blocks.
struct MoeUnit {
  int e, m0, n0, row_end, r0, kb;
};
// The unit that worker `w` of `n` takes in its round that starts at `base`.  The weight GEMMs' units cost as much as
// their experts have rows; they stand in falling order, and every other round is dealt backwards, so that the workers'
// sums come out nearly even.  (In the experts' order one pair of CTAs had up to 1.3 times the mean, 16 experts with
// 1,800 to 7,900 rows, 768 x 1536: forward and backward 1111-1116 us in five long runs, in this one 1079-1090 in five
// between them.)
template <int MODE>
__device__ __forceinline__ int unit_of(int base, int w, int n) {
  return base + (MODE == MOE_DW && (base / n & 1) ? n - 1 - w : w);
}
template <int MODE, int BM, int BN>
__device__ __forceinline__ MoeUnit moe_unit(const MoeGemmArgs& a, int u, int mt, int nt) {
  MoeUnit q;
  int mi, ni;
  if (MODE == MOE_DW) {
    const int o = u / (mt * nt);
    q.e = __ldcg(a.order + o);
    tile_coords(u - o * mt * nt, mt, nt, mi, ni);
    q.m0 = mi * BM;
    q.row_end = a.M;
    q.r0 = __ldcg(a.off + q.e);
    q.kb = (__ldcg(a.off + q.e + 1) - q.r0) / kBK;
  } else {
    tile_coords(u, mt, nt, mi, ni);
    const int4 t = __ldcg(a.tile + mi);
    q.e = t.x;
    q.m0 = t.y;
    q.row_end = t.z;
    q.r0 = 0;
    q.kb = (a.K + kBK - 1) / kBK;
  }
  q.n0 = ni * BN;
  return q;
}

// Two fp32 operations an instruction: in an epilogue with an activation a warp's arithmetic is most of a chunk's time
// (a 32x32 chunk of dpre took 1,100 instructions with scalar ones; its GEMM 198 us, with these 179).
__device__ __forceinline__ uint64_t f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_get(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2s(float a) { return f2(a, a); }
constexpr float kGeluC = 0.7978845608028654f;       // sqrt(2 / pi)
constexpr float kGeluC3 = kGeluC * 0.044715f;
// t = tanh(c x + c3 x^3), two at a time; x2 = x^2
__device__ __forceinline__ uint64_t gelu_tanh2(uint64_t x, uint64_t x2) {
  float a, b;
  f2_get(mul2(x, fma2(x2, f2s(kGeluC3), f2s(kGeluC))), a, b);
  return f2(tanh_fast(a), tanh_fast(b));
}
__device__ __forceinline__ uint64_t gelu2(uint64_t x) {  // x / 2 (1 + t)
  const uint64_t h = mul2(x, f2s(0.5f));
  return fma2(h, gelu_tanh2(x, mul2(x, x)), h);
}
// act = x / 2 (1 + t), slope = (1 + t) / 2 + x / 2 (1 - t^2) (c + 3 c3 x^2)
__device__ __forceinline__ void gelu_both2(uint64_t x, uint64_t& act, uint64_t& slope) {
  const uint64_t x2 = mul2(x, x);
  const uint64_t t = gelu_tanh2(x, x2);
  const uint64_t hx = mul2(x, f2s(0.5f));
  act = fma2(hx, t, hx);
  const uint64_t r = mul2(hx, fma2(x2, f2s(3.f * kGeluC3), f2s(kGeluC)));
  const uint64_t w = fma2(mul2(t, f2s(-1.f)), t, f2s(1.f));
  slope = fma2(r, w, fma2(t, f2s(0.5f), f2s(0.5f)));
}

__device__ __forceinline__ float row_gate(const MoeGemmArgs& a, int row) {
  if (a.gates == nullptr) return 1.f;
  const int s = __ldcg(a.src + row);
  if (s < 0) return 0.f;
  return a.gates_f32 ? reinterpret_cast<const float*>(a.gates)[s] : bf2f(reinterpret_cast<const bf16*>(a.gates)[s]);
}

// Unpack this lane's 64-byte row of a slab to fp32.
__device__ __forceinline__ void slab_get_bf16(const uint8_t* slab, int lane, float* v) {
  const uint4* src = reinterpret_cast<const uint4*>(slab + lane * 64);
#pragma unroll
  for (int j = 0; j < 4; ++j) unpack8(src[slab_unit_bf16(lane, j)], v + 8 * j);
}

// What a role still has in flight when it leaves its loop, also by a wait that ran out: loads that would land in, and
// products that would read from and signal to, a CTA that is gone.  Both wait (mbar_wait's limit; the CTA's abort flag
// does not shorten it) until that is done.  `stage` and `phase`: where the ring goes next, so a stage before it was
// last used in this pass over the ring, the others in the pass before (which a fresh barrier counts as complete).
template <int STAGES>
__device__ __forceinline__ void finish_loads(uint64_t* full_bar, int stage, uint32_t phase) {
  volatile int never = 0;
  for (int s = 0; s < STAGES; ++s) mbar_wait(&full_bar[s], s < stage ? phase : phase ^ 1, &never);
}
template <int STAGES>
__device__ __forceinline__ void finish_products(uint64_t* empty_bar, int stage, uint32_t phase) {
  volatile int never = 0;  // products complete in order: the last stage's
  mbar_wait(&empty_bar[stage ? stage - 1 : STAGES - 1], stage ? phase : phase ^ 1, &never);
}

// One 32x32 chunk: this lane's row of 32 accumulators -> slab -> TMA store.  `staged` (MOE_DGELU): the chunk's
// pre-activations, already in shared memory; null: read from global memory.
__device__ __forceinline__ void moe_epi_chunk(const MoeGemmArgs& a, const CUtensorMap* tmOut, const CUtensorMap* tmAux,
                                              uint8_t* slab, int lane, int row0, int col, int e, bool dw, float* v,
                                              float gate, float& dot, const uint8_t* staged) {
  switch (a.epi) {
    case MOE_PLAIN:
    case MOE_GELU: {
      if (a.bias) {
        float b[32];
        load_row32(a.bias + (long)e * a.N, col, a.N, b);
#pragma unroll
        for (int j = 0; j < 32; j += 2)
          f2_get(fma2(f2s(a.epi == MOE_PLAIN ? gate : 1.f), f2(b[j], b[j + 1]), f2(v[j], v[j + 1])), v[j], v[j + 1]);
      }
      if (a.epi == MOE_GELU) {
        if (a.save_aux) slab_put_bf16(slab + 2048, lane, v);
#pragma unroll
        for (int j = 0; j < 32; j += 2) f2_get(mul2(f2s(gate), gelu2(f2(v[j], v[j + 1]))), v[j], v[j + 1]);
      }
      slab_put_bf16(slab, lane, v);
      break;
    }
    case MOE_DGELU: {
      float h[32];
      if (staged) slab_get_bf16(staged, lane, h);
      else load_row32(a.aux_in + (long)(row0 + lane) * a.N, col, a.N, h);
      uint64_t d2 = 0;
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        uint64_t act, slope;
        const uint64_t acc = f2(v[j], v[j + 1]);
        gelu_both2(f2(h[j], h[j + 1]), act, slope);
        d2 = fma2(acc, act, d2);
        f2_get(mul2(mul2(f2s(gate), acc), slope), v[j], v[j + 1]);
      }
      float da, db;
      f2_get(d2, da, db);
      dot += da + db;
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
  if (a.epi == MOE_DGELU && a.sums != nullptr) {
    // lane: two columns of every other row, from the slab (as rounded); the two row halves meet in lanes 0-15
    const int cp = lane & 15, h = lane >> 4;
    uint64_t acc = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = 2 * i + h;
      const uint32_t w = *reinterpret_cast<const uint32_t*>(slab + r * 64 + slab_unit_bf16(r, cp >> 2) * 16 + (cp & 3) * 4);
      acc = add2(acc, f2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)));
    }
    float s0, s1;
    f2_get(acc, s0, s1);
    s0 += __shfl_xor_sync(0xffffffffu, s0, 16);
    s1 += __shfl_xor_sync(0xffffffffu, s1, 16);
    if (h == 0 && col + 2 * cp < a.N)
      *reinterpret_cast<float2*>(a.sums + (long)(row0 >> 5) * a.N + col + 2 * cp) = make_float2(s0, s1);
  }
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
  pdl_wait();
  pdl_launch();

  const int nt = (args.N + BN - 1) / BN;
  const int mt = MODE == MOE_DW ? (args.M + kBM - 1) / kBM : __ldcg(args.ntile);
  const int units = MODE == MOE_DW ? args.E * mt * nt : mt * nt;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------------ TMA producer
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int base = 0; base < units && ok; base += gridDim.x) {
        const int u = unit_of<MODE>(base, blockIdx.x, gridDim.x);
        if (u >= units) continue;
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
      finish_loads<Cfg::STAGES>(full_bar, stage, phase);
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
      for (int base = 0; base < units && ok; base += gridDim.x) {
        const int u = unit_of<MODE>(base, blockIdx.x, gridDim.x);
        if (u >= units) continue;
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
      finish_products<Cfg::STAGES>(empty_bar, stage, phase);
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
    for (int base = 0; base < units; base += gridDim.x) {
      const int u = unit_of<MODE>(base, blockIdx.x, gridDim.x);
      if (u >= units) continue;
      const MoeUnit q = moe_unit<MODE, kBM, BN>(args, u, mt, nt);
      if (q.kb > 0) {
        if (!mbar_wait(&tfull_bar[ab], aphase, abort_flag)) break;
        tc_fence_after();
      }
      const int row0 = q.m0 + q4 * 32;
      const uint32_t tbase = tmem_base + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(ab * BN);
      const int c_begin = half * (BN / 2), c_end = c_begin + BN / 2;
      if (row0 < q.row_end) {  // rows of the next expert (or past the matrix) are not this tile's
        const float gate = MODE == MOE_DW ? 1.f : row_gate(args, row0 + lane);
        float dot = 0.f;
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
                        MODE == MOE_DW, v, gate, dot, nullptr);
          ++ck;
        }
        if (MODE == MOE_DX && args.dots != nullptr)
          args.dots[(long)(q.n0 / (BN / 2) + half) * args.R + row0 + lane] = dot;
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

// -------------------------------------------------------------------------
// 2-SM variant: a cluster of two CTAs computes a 256x256 tile (tcgen05 cta_group::2).
// CTA r loads its 128 rows of A and its 128 columns of B (32 KB a k-block where the 1-SM
// 128x256 tile loads 48 KB, for half the output), the leader issues the MMAs of both.
// Barriers as in the dense pair GEMM (gemm.cu): full (leader; both CTAs' bytes), empty and
// tile-full (both, by the leader's commit), tile-empty (leader; both epilogues), done.
// No load is multicast.
//
// Bound: at K 2048 by the tensor cores at the power limit (32768 rows x 2048 x 2048: 218 us a
// product, 1.26 PFLOP/s, with an eighth of the tiles' rows padding; the dense pair GEMM of the
// same size 190).  At K 768 the products with an activation take 153 us forward and 179 backward
// (65536 rows x 1536) where one without takes 112.  No unit is full there (counters at 32768 rows,
// forward / backward: tensor pipe 43 / 36%, issue 28 / 36%, DRAM 31 / 29%).  The likely bound, not
// shown, is the chain in each epilogue warp: a chunk is read from TMEM, computed, packed and handed
// to its store before the next one is read.  Twice the epilogue warps (96 registers) were no faster.
__device__ __forceinline__ void tma_load_3d_pair(const CUtensorMap* map, void* dst, uint32_t leader_bar, int x, int y,
                                                 int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(leader_bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

struct MoePairCfg {
  static constexpr int A_BYTES = kBM * kBK * 2;
  static constexpr int B_BYTES = 128 * kBK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 5;
  static constexpr int TMEM_COLS = 512;
  static constexpr int EPI_BYTES = kEpiWarps * 2 * kEpiSlab;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_BYTES + 1024 /*align*/ + 256 /*barriers: 15 + 16, and two words*/;
  static_assert((2 * STAGES + 5 + 2 * kEpiWarps) * 8 + 8 <= 256, "barriers");
};

template <int MODE>
__global__ void __maxnreg__(DTB_CORESIDENT_MAXNREG)
    moe_gemm2_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ CUtensorMap tmAux,
                     MoeGemmArgs args) {
  using Cfg = MoePairCfg;
  constexpr bool A_MN = MODE == MOE_DW, B_MN = MODE != MOE_DX;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi_smem = smem + Cfg::STAGES * Cfg::STAGE_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(epi_smem + Cfg::EPI_BYTES);
  uint64_t* empty_bar = full_bar + Cfg::STAGES;
  uint64_t* tfull_bar = empty_bar + Cfg::STAGES;  // [2]
  uint64_t* tempty_bar = tfull_bar + 2;           // [2]
  uint64_t* done_bar = tempty_bar + 2;
  uint64_t* aux_bar = done_bar + 1;  // [epilogue warps][2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(aux_bar + 2 * kEpiWarps);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull_bar[b], 1);
      mbar_init(&tempty_bar[b], 2 * kEpiWarps);
    }
    mbar_init(done_bar, 1);
    for (int b = 0; b < 2 * kEpiWarps; ++b) mbar_init(&aux_bar[b], 1);
    *abort_flag = 0;
    fence_barrier_init_cluster();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, Cfg::TMEM_COLS);
  tc_fence_before();
  cluster_sync_all();  // both CTAs' barriers initialised and TMEM allocated
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  pdl_launch();

  const int nt = (args.N + 255) / 256;
  const int mt = MODE == MOE_DW ? (args.M + 255) / 256 : __ldcg(args.ntile);
  const int units = MODE == MOE_DW ? args.E * mt * nt : mt * nt;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------------------ TMA producer (both CTAs)
      const uint32_t lead_full0 = mapa_shared(&full_bar[0], 0);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int base = 0; base < units && ok; base += npairs) {
        const int u = unit_of<MODE>(base, pair, npairs);
        if (u >= units) continue;
        const MoeUnit q = moe_unit<MODE, 256, 256>(args, u, mt, nt);
        const int m0 = q.m0 + (int)rank * 128, n0 = q.n0 + (int)rank * 128;
        for (int kb = 0; kb < q.kb; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag)) { ok = false; break; }
          uint8_t* sA = smem + stage * Cfg::STAGE_BYTES;
          uint8_t* sB = sA + Cfg::A_BYTES;
          const uint32_t fb = lead_full0 + (uint32_t)(stage * sizeof(uint64_t));
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2 * Cfg::STAGE_BYTES);
          if (MODE == MOE_DW) {
            const int r0 = q.r0 + kb * kBK;
            tma_load_2d_pair(&tmA, sA, fb, m0, r0);
            tma_load_2d_pair(&tmA, sA + 8192, fb, m0 + 64, r0);
            tma_load_2d_pair(&tmB, sB, fb, n0, r0);
            tma_load_2d_pair(&tmB, sB + 8192, fb, n0 + 64, r0);
          } else {
            const int k0 = kb * kBK;
            tma_load_2d_pair(&tmA, sA, fb, k0, m0);
            if (MODE == MOE_DX) {
              tma_load_3d_pair(&tmB, sB, fb, k0, n0, q.e);
            } else {
              tma_load_3d_pair(&tmB, sB, fb, n0, k0, q.e);
              tma_load_3d_pair(&tmB, sB + 8192, fb, n0 + 64, k0, q.e);
            }
          }
          if (++stage == Cfg::STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // Both CTAs' loads are counted on the leader's barriers.  The other one, should a wait have run out here, gives
      // its own a millisecond.
      if (leader) {
        finish_loads<Cfg::STAGES>(full_bar, stage, phase);
      } else if (!ok) {
        for (const uint64_t t0 = globaltimer_ns(); globaltimer_ns() - t0 < 1000000;) {}
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // ------------------------------------------------------------ MMA issuer (leader only)
      constexpr uint32_t idesc = make_idesc_bf16(256, 256, A_MN, B_MN);
      int stage = 0;
      uint32_t phase = 0;
      int ab = 0;
      uint32_t aphase = 0;
      bool ok = true;
      for (int base = 0; base < units && ok; base += npairs) {
        const int u = unit_of<MODE>(base, pair, npairs);
        if (u >= units) continue;
        const MoeUnit q = moe_unit<MODE, 256, 256>(args, u, mt, nt);
        if (q.kb == 0) continue;  // an expert without rows: the epilogue writes zeros
        if (!mbar_wait(&tempty_bar[ab], aphase ^ 1, abort_flag)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(ab * 256);
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
            tc_mma_f16_pair(d_tmem, ad, bd, idesc, (kb > 0 || kk > 0) ? 1u : 0u);
          }
          tc_commit_pair(&empty_bar[stage], 0x3);
          if (++stage == Cfg::STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tc_commit_pair(&tfull_bar[ab], 0x3);
        if (++ab == 2) { ab = 0; aphase ^= 1; }
      }
      finish_products<Cfg::STAGES>(empty_bar, stage, phase);
    }
  } else {
    // -------------------------------------------------------------- epilogue (both CTAs)
    const int ew = warp - 2;
    const int q4 = warp & 3;
    const int half = ew >> 2;
    uint8_t* slab = epi_smem + ew * 2 * kEpiSlab;
    uint64_t* abar = aux_bar + ew * 2;
    const uint32_t lead_tempty0 = mapa_shared(&tempty_bar[0], 0);
    // MOE_DGELU: a chunk's pre-activations come by TMA into the second half of its slab, two chunks ahead and
    // the tile's first two before its products are done.  (The dpre GEMM of 65536 rows x 1536, K 768, took 224 us
    // with the lanes reading a row each and scalar arithmetic, 198 with TMA, 179 with two operations an instruction.)
    const bool stage_aux = MODE == MOE_DX && args.epi == MOE_DGELU;
    volatile int never = 0;  // these copies are waited for whatever the abort flag says: none stays in flight
    uint32_t ck = 0;
    int ab = 0;
    uint32_t aphase = 0;
    for (int base = 0; base < units; base += npairs) {
      const int u = unit_of<MODE>(base, pair, npairs);
      if (u >= units) continue;
      const MoeUnit q = moe_unit<MODE, 256, 256>(args, u, mt, nt);
      const int row0 = q.m0 + (int)rank * 128 + q4 * 32;
      const int c0 = q.n0 + half * 128;
      // chunks of 32 columns that this warp has to do (none where its rows are not this tile's)
      const int chunks = row0 < q.row_end ? max(0, min(4, (args.N - c0 + 31) / 32)) : 0;
      if (stage_aux && lane == 0) {
        fence_proxy_async_smem();
        for (int i = 0; i < min(2, chunks); ++i) {
          const uint32_t b = (ck + i) & 1;
          mbar_arrive_expect_tx(&abar[b], 2048);
          tma_load_2d(&tmAux, slab + b * kEpiSlab + 2048, &abar[b], c0 + 32 * i, row0);
        }
      }
      if (q.kb > 0) {
        if (!mbar_wait(&tfull_bar[ab], aphase, abort_flag)) {
          if (stage_aux) {
            for (int i = 0; i < min(2, chunks); ++i) mbar_wait(&abar[(ck + i) & 1], ((ck + i) >> 1) & 1, &never);
          }
          break;
        }
        tc_fence_after();
      }
      const uint32_t tbase = tmem_base + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(ab * 256 + half * 128);
      const float gate = MODE == MOE_DW || row0 >= q.row_end ? 1.f : row_gate(args, row0 + lane);
      float dot = 0.f;
#pragma unroll 1
      for (int i = 0; i < chunks; ++i) {
        uint8_t* sl = slab + (ck & 1) * kEpiSlab;
        float v[32];
        if (q.kb > 0) {
          tmem_ld32(tbase + 32 * i, v);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0.f;
        }
        epi_slab_acquire(lane, true);
        if (stage_aux) mbar_wait(&abar[ck & 1], (ck >> 1) & 1, &never);
        moe_epi_chunk(args, &tmOut, &tmAux, sl, lane, row0, c0 + 32 * i, q.e, MODE == MOE_DW, v, gate,
                      dot, stage_aux ? sl + 2048 : nullptr);
        if (stage_aux && i + 2 < chunks && lane == 0) {  // every lane has read the buffer (moe_epi_chunk synchronises)
          mbar_arrive_expect_tx(&abar[ck & 1], 2048);
          tma_load_2d(&tmAux, sl + 2048, &abar[ck & 1], c0 + 32 * (i + 2), row0);
        }
        ++ck;
      }
      if (MODE == MOE_DX && args.dots != nullptr && row0 < q.row_end)
        args.dots[(long)(q.n0 / 128 + half) * args.R + row0 + lane] = dot;
      if (q.kb > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(lead_tempty0 + (uint32_t)(ab * sizeof(uint64_t)));
        if (++ab == 2) { ab = 0; aphase ^= 1; }
      }
    }
    if (lane == 0) bulk_wait0();
    __syncwarp();
  }

  // Neither CTA releases the pair's TMEM before the other has finished with it.
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) {
    mbar_arrive_cluster(mapa_shared(done_bar, rank ^ 1));
    mbar_wait(done_bar, 0, abort_flag);
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
  }
}

// -------------------------------------------------------------------------
// Forward products for few rows an expert (generation with a batch): 64-row tiles with the
// operands swapped, out^T = W_e^T . rows^T.  The weights' 128 columns are the M side of the
// tile (MN-major), up to 64 rows the N side, so a k-block is 16 KB of weights and 8 KB of
// rows instead of 32 KB and 16 KB for rows that are mostly padding; two or three CTAs an SM
// keep about 200 KB in flight.  A CTA makes one tile over one part of K: the first product all of it,
// with the activation; the second leaves fp32 parts that moe_thin_combine joins.  Bound by
// the weights' way from DRAM and five launches in a row: 48 tokens x 2 of 8 experts, 1024 x 4096
// (134 MB of weights, 20.4 us at the copy rate), take 39 us in all, with the 128-row tiles 69.
// (Asking for all of a CTA's weights in L2 at its start made that 42.)
template <int S>
struct MoeThinCfg {
  static constexpr int A_BYTES = 128 * kBK * 2;
  static constexpr int B_BYTES = kRowPad * kBK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = S;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 /*align*/ + 128 /*barriers*/;
};
constexpr int kThinThreads = 192;
struct MoeThinArgs {
  const int4* tile;
  const int* off;
  int E, N, K, splits;
  const bf16* bias;  // act: [E, N] or null
  bf16* act;         // [R, N] = gelu(acc + bias), or
  float* part;       // [splits, R, N] = acc
  long R;
};

// The plan is complete before this kernel can start (its predecessor has waited for it), so only the rows are waited for.
template <int S>
__global__ void __launch_bounds__(kThinThreads)
    moe_thin_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, MoeThinArgs a) {
  using Cfg = MoeThinCfg<S>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + Cfg::STAGES * Cfg::STAGE_BYTES);
  uint64_t* empty_bar = full_bar + Cfg::STAGES;
  uint64_t* done_bar = empty_bar + Cfg::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
  }
  if (warp == 1) tmem_alloc(tmem_slot, kRowPad);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  const int nt = (a.N + 127) / 128;
  const int per = nt * a.splits;
  const int ti = blockIdx.x / per, ni = blockIdx.x % per / a.splits, sp = blockIdx.x % a.splits;
  const bool there = ti < __ldcg(a.off + a.E) / kRowPad;
  if (there) {
    const int4 t = __ldcg(a.tile + ti);
    const int n0 = ni * 128;
    const int kbs = (a.K + kBK - 1) / kBK;
    const int kb0 = (int)((long)kbs * sp / a.splits), kb1 = (int)((long)kbs * (sp + 1) / a.splits);
    if (warp == 0) {
      if (lane == 0) {
        const auto weights = [&](int stage, int kb) {
          uint8_t* sA = smem + stage * Cfg::STAGE_BYTES;
          mbar_arrive_expect_tx(&full_bar[stage], Cfg::STAGE_BYTES);
          tma_load_3d(&tmW, sA, &full_bar[stage], n0, kb * kBK, t.x);
          tma_load_3d(&tmW, sA + 8192, &full_bar[stage], n0 + 64, kb * kBK, t.x);
        };
        // the first weights come while the rows are still being made
        const int first = min(kb1 - kb0, Cfg::STAGES);
        for (int i = 0; i < first; ++i) weights(i, kb0 + i);
        pdl_wait();
        pdl_launch();
        int stage = 0;
        uint32_t phase = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (kb - kb0 >= Cfg::STAGES) {
            if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag)) break;
            weights(stage, kb);
          }
          tma_load_2d(&tmX, smem + stage * Cfg::STAGE_BYTES + Cfg::A_BYTES, &full_bar[stage], kb * kBK, t.y);
          if (++stage == Cfg::STAGES) { stage = 0; phase ^= 1; }
        }
        finish_loads<Cfg::STAGES>(full_bar, stage, phase);
      }
    } else if (warp == 1) {
      if (lane == 0) {
        constexpr uint32_t idesc = make_idesc_bf16(128, kRowPad, true, false);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint32_t aBase = smem_u32(smem + stage * Cfg::STAGE_BYTES);
          const uint32_t bBase = aBase + Cfg::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk)
            tc_mma_f16(tmem, make_sw128_desc(aBase + kk * 2048, 8192, 1024), make_sw128_desc(bBase + kk * 32, 16, 1024),
                       idesc, (kb > kb0 || kk > 0) ? 1u : 0u);
          tc_commit(&empty_bar[stage]);
          if (++stage == Cfg::STAGES) { stage = 0; phase ^= 1; }
        }
        if (ok) tc_commit(done_bar);
        finish_products<Cfg::STAGES>(empty_bar, stage, phase);
      }
    } else {
      // lane = a column of the output, TMEM column = a row
      const int col = n0 + (warp & 3) * 32 + lane;
      const int rows = min(kRowPad, t.z - t.y);
      if (mbar_wait(done_bar, 0, abort_flag)) {
        tc_fence_after();
        const float b = a.bias && col < a.N ? bf2f(a.bias[(long)t.x * a.N + col]) : 0.f;
#pragma unroll 1
        for (int h = 0; h < kRowPad; h += 32) {
          if (h >= rows) break;
          float v[32];
          tmem_ld32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + h, v);
          if (col < a.N) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              if (h + j >= rows) break;
              if (a.act) a.act[(long)(t.y + h + j) * a.N + col] = f2bf(gelu_fast(v[j] + b));
              else a.part[((long)sp * a.R + t.y + h + j) * a.N + col] = v[j];
            }
          }
        }
      }
    }
  }
  if (threadIdx.x == 0) pdl_wait();  // CTAs without a tile too: none is done before the rows are
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kRowPad);
  }
}

// y[n] = sum_j gate_j (sum of the row's parts + b2_e): a thread per four columns.
template <typename I, typename G>
__global__ void __launch_bounds__(128)
    moe_thin_combine_kernel(const float* __restrict__ part, const bf16* __restrict__ b2, const I* __restrict__ idx,
                            const G* __restrict__ gates, bf16* __restrict__ y, MoePlan pl, int E, int Co, int k,
                            int splits, long R) {
  pdl_wait();
  const long n = blockIdx.x;
  const int c = (blockIdx.y * 128 + threadIdx.x) * 4;
  if (c >= Co) return;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j = 0; j < k; ++j) {
    const int r = __ldcg(pl.inv + n * k + j);
    if (r < 0) continue;
    const float g = load_gate(gates, n * k + j);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int p = 0; p < splits; ++p) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(part + ((long)p * R + r) * Co + c));
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    if (b2) {
      const bf16* b = b2 + (long)slot_expert(idx, n * k + j, E) * Co + c;
      s.x += bf2f(b[0]); s.y += bf2f(b[1]); s.z += bf2f(b[2]); s.w += bf2f(b[3]);
    }
    acc.x = fmaf(g, s.x, acc.x); acc.y = fmaf(g, s.y, acc.y); acc.z = fmaf(g, s.z, acc.z); acc.w = fmaf(g, s.w, acc.w);
  }
  *reinterpret_cast<uint2*>(y + n * Co + c) = make_uint2(pack_bf16x2(acc.x, acc.y), pack_bf16x2(acc.z, acc.w));
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

// Programmatic dependent launch of `kern` on `st` (common shape of the launches below).
template <typename... Args, typename... Given>
static void launch_pdl(void (*kern)(Args...), dim3 grid, int threads, int smem, cudaStream_t st, Given&&... given) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, Args(given)...));
  count_launch();
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
  launch_pdl(kern, dim3(grid), kThreads, MoeCfg<BN>::SMEM_BYTES, st, ta, tb, to, tx, a);
}

// Pairs that can be resident at once.
static int moe_max_pairs() {
  static int n = -1;
  if (n < 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (num_sms() / 2), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = MoePairCfg::SMEM_BYTES;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaFuncSetAttribute(moe_gemm2_kernel<MOE_FWD>, cudaFuncAttributeMaxDynamicSharedMemorySize, MoePairCfg::SMEM_BYTES);
    int c = 0;
    if (cudaOccupancyMaxActiveClusters(&c, moe_gemm2_kernel<MOE_FWD>, &cfg) != cudaSuccess || c <= 0) {
      cudaGetLastError();
      c = num_sms() / 2;
    }
    n = c;
  }
  return n;
}

template <int MODE>
static void launch_moe2(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& to, const CUtensorMap& tx,
                        const MoeGemmArgs& a, long units, cudaStream_t st) {
  static bool attr_set = false;
  auto kern = moe_gemm2_kernel<MODE>;
  if (!attr_set) {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, MoePairCfg::SMEM_BYTES);
    attr_set = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (unsigned)std::min<long>(units, moe_max_pairs()), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = MoePairCfg::SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, ta, tb, to, tx, a));
  count_launch();
}

struct MoeSizes {
  long n, k, P, E, R;  // tokens, slots a token, slots, experts, most padded rows
};

// What a grouped GEMM has beside its operands.
struct MoeExtra {
  int epi = MOE_PLAIN;
  const bf16* bias = nullptr;
  bf16* aux = nullptr;     // MOE_GELU: written, MOE_DGELU: read
  float* sums = nullptr;
  float* dots = nullptr;
  const at::Tensor* gates = nullptr;
};
static MoeGemmArgs moe_args(const MoeExtra& x, const MoePlan& pl, const MoeSizes& z) {
  MoeGemmArgs g{};
  g.off = pl.off;
  g.order = pl.order;
  g.E = (int)z.E;
  g.epi = x.epi;
  g.bias = x.bias;
  g.aux_in = x.aux;
  g.save_aux = x.epi == MOE_GELU && x.aux != nullptr;
  g.sums = x.sums;
  g.dots = x.dots;
  g.R = z.R;
  g.src = pl.src;
  if (x.gates) {
    g.gates = x.gates->const_data_ptr();
    g.gates_f32 = x.gates->scalar_type() == at::kFloat;
  }
  return g;
}

struct MoeTiling {
  bool pair;  // 256 x 256 by a CTA pair
  int bn;     // else 128 x bn
};
// 256-row pair tiles once the experts have 256 rows on average (below, half of a tile is padding).  Pairs against
// 1-SM tiles, 16 experts 2048 x 2048, forward, 256 / 512 / 1024 / 2048 rows each: 118 / 178 / 289 / 533 us
// (129 / 174 / 302 / 562).  Where 256-wide tiles do not fill the SMs, 128 x 128: forward and
// backward in a CUDA graph, 4 experts 768 x 1536, 600 tokens, two a token, 82 us (256-wide 93); 8 experts 512 x 1024,
// 2048 tokens, 107 (111).
static MoeTiling moe_rows_tiling(int N, const MoeSizes& z) {
  if (N <= 128 || (z.P / 256 + std::min(z.P, z.E)) * ((N + 255) / 256) < num_sms() / 2) return {false, 128};
  return {z.P >= 256 * z.E, 256};
}
static MoeTiling moe_weight_tiling(int M, int N, const MoeSizes& z) {
  if (N <= 128 || z.E * ((M + 255) / 256) * ((N + 255) / 256) < num_sms() / 2) return {false, 128};
  return {M > 128, 256};
}
// The tiles of a training call's products: up (and dpre), down, dx, dw1, dw2.
std::vector<std::string> experts_tiles(int64_t n, int64_t k, int64_t E, int64_t C, int64_t H, int64_t Co) {
  const MoeSizes z{n, k, n * k, E, moe_max_rows(n * k, E)};
  const auto name = [](const MoeTiling& t) {
    return t.pair ? std::string("256x256 pair") : "128x" + std::to_string(t.bn);
  };
  return {name(moe_rows_tiling((int)H, z)), name(moe_rows_tiling((int)Co, z)), name(moe_rows_tiling((int)C, z)),
          name(moe_weight_tiling((int)C, (int)H, z)), name(moe_weight_tiling((int)H, (int)Co, z))};
}
// Parts of each row's product that the dpre GEMM leaves.
static int moe_dot_parts(int N, const MoeSizes& z) {
  const int bn = moe_rows_tiling(N, z).bn;
  return (N + bn - 1) / bn * 2;
}

// rows [R, N] = rows [R, K] . W_e (MOE_FWD, w [E, K, N]) or . W_e^T (MOE_DX, w [E, N, K])
static void moe_rows_gemm(int mode, const bf16* a, const bf16* w, bf16* out, int N, int K, const MoeExtra& x,
                          const MoePlan& pl, const MoeSizes& z, cudaStream_t st) {
  const MoeTiling t = moe_rows_tiling(N, z);
  const bool pair = t.pair;
  MoeGemmArgs g = moe_args(x, pl, z);
  g.tile = pair ? pl.tile2 : pl.tile;
  g.ntile = pl.ntile + (pair ? 1 : 0);
  g.N = N;
  g.K = K;
  g.M = 1;
  const int bn = t.bn;
  const CUtensorMap ta = make_map(a, z.R, K, K, 64, kBM);
  const CUtensorMap tb = mode == MOE_FWD ? make_map3(w, z.E, K, N, 64, 64) : make_map3(w, z.E, N, K, 64, pair ? 128 : bn);
  const CUtensorMap to = make_store_map(out, false, z.R, N, N);
  const CUtensorMap tx = x.aux ? make_store_map(x.aux, false, z.R, N, N) : to;
  const long units = moe_max_tiles(z.P, z.E) * ((N + bn - 1) / bn);
  if (pair) {
    if (mode == MOE_FWD) launch_moe2<MOE_FWD>(ta, tb, to, tx, g, units, st);
    else launch_moe2<MOE_DX>(ta, tb, to, tx, g, units, st);
  } else if (mode == MOE_FWD) {
    if (bn == 256) launch_moe<256, MOE_FWD>(ta, tb, to, tx, g, units, st);
    else launch_moe<128, MOE_FWD>(ta, tb, to, tx, g, units, st);
  } else {
    if (bn == 256) launch_moe<256, MOE_DX>(ta, tb, to, tx, g, units, st);
    else launch_moe<128, MOE_DX>(ta, tb, to, tx, g, units, st);
  }
}

// out_e [M, N] (fp32 or bf16) = a_e^T . b_e over the expert's rows
static void moe_weight_gemm(const bf16* a, const bf16* b, const at::Tensor& out, int M, int N, const MoePlan& pl,
                            const MoeSizes& z, cudaStream_t st) {
  const bool f32 = out.scalar_type() == at::kFloat;
  MoeExtra x;
  x.epi = f32 ? MOE_F32 : MOE_PLAIN;
  MoeGemmArgs g = moe_args(x, pl, z);
  g.M = M;
  g.N = N;
  const MoeTiling t = moe_weight_tiling(M, N, z);
  const int bn = t.bn;
  const CUtensorMap ta = make_map(a, z.R, M, M, 64, 64);
  const CUtensorMap tb = make_map(b, z.R, N, N, 64, 64);
  const CUtensorMap to = make_store_map(out.data_ptr(), f32, M, N, N, z.E);
  if (t.pair) {
    launch_moe2<MOE_DW>(ta, tb, to, to, g, z.E * ((M + 255) / 256) * ((N + 255) / 256), st);
    return;
  }
  const long units = z.E * ((M + kBM - 1) / kBM) * ((N + bn - 1) / bn);
  if (bn == 256) launch_moe<256, MOE_DW>(ta, tb, to, to, g, units, st);
  else launch_moe<128, MOE_DW>(ta, tb, to, to, g, units, st);
}

static int warp_grid(long rows) { return (int)std::max<long>(1, std::min<long>((rows + 7) / 8, 148L * 8)); }

template <typename I>
static void moe_build_plan_of(const I* idx, const MoePlan& pl, const MoeSizes& z, cudaStream_t st) {
  const int nb = (int)plan_blocks(z.P), E = (int)z.E;
  if (z.P <= kPlanSmall) {
    moe_plan_kernel<I><<<1, kMoeMaxExperts, kMoeMaxExperts / 32 * E * 4, st>>>(idx, (int)z.P, E, pl);
    count_launch();
  } else {
    moe_hist_kernel<I><<<nb, kPlanThreads, E * 4, st>>>(idx, z.P, E, pl);
    count_launch();
    launch_pdl(moe_offsets_kernel, dim3(1), kMoeMaxExperts, 0, st, nb, E, pl);
    launch_pdl(moe_place_kernel<I>, dim3(nb), kPlanThreads, 8 * E * 4, st, idx, z.P, E, pl);
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}
static void moe_build_plan(const at::Tensor& idx, const MoePlan& pl, const MoeSizes& z, cudaStream_t st) {
  if (idx.scalar_type() == at::kInt) moe_build_plan_of(idx.data_ptr<int>(), pl, z, st);
  else moe_build_plan_of(reinterpret_cast<const long*>(idx.data_ptr<int64_t>()), pl, z, st);
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

// Up to this many slots go the streaming way: each slot reads its expert's weights, so it loses once many slots share
// experts.  Streaming against the 64-row tiles, in a CUDA graph with cold weights, two slots a token:
//   1 token  of 16 experts 768 x 2048: 10.3 / 19.3 us,  of 8 experts 1024 x 4096: 15.5 / 26.7 us
//   4 tokens                           18.7 / 26.0                                28.0 / 31.3
//   8 tokens                           28.6 / 29.3                                49.4 / 34.8
constexpr long kFewSlots = 8;
// Up to this many rows an expert on average, the 64-row tiles; past it most experts need a second one.  Against the
// 128-row tiles, in a CUDA graph with cold weights: 8 experts 1024 x 4096, 32 / 64 / 96 / 128 rows each on average,
// 40 / 43 / 60 / 64 us (61 / 62 / 67 / 68); 32 experts 768 x 1536, 64 / 96 / 128 rows, 57 / 64 / 83 us (60 / 61 / 64).
constexpr long kThinRows = 64;

template <typename I, typename G>
static void moe_few_launch(const bf16* x, const bf16* w1, const bf16* b1, const bf16* w2, const bf16* b2, const I* idx,
                           const G* gates, float* h, bf16* y, int C, int H, int Co, const MoeSizes& z, cudaStream_t st) {
  const int E = (int)z.E, k = (int)z.k;
  // the most column vectors a row (whole lines, fewer CTAs to join) that still give every SM a CTA
  const auto lanes = [](long cols, long per) {
    for (int l = 16; l > 4; l /= 2)
      if ((cols + 8 * l - 1) / (8 * l) * per >= num_sms()) return l;
    return 4;
  };
  const int l1 = lanes(H, z.P), l2 = lanes(Co, z.n * kFewCluster);
#define DTB_FEW_UP(L)                                                                                              \
  moe_few_up_kernel<I, L><<<dim3((H + 8 * L - 1) / (8 * L), (unsigned)z.P), kFewThreads, C * 4, st>>>(x, w1, b1, idx, h, E, \
                                                                                                     C, H, k)
  if (l1 == 16) DTB_FEW_UP(16);
  else if (l1 == 8) DTB_FEW_UP(8);
  else DTB_FEW_UP(4);
#undef DTB_FEW_UP
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kFewCluster, (unsigned)((Co + 8 * l2 - 1) / (8 * l2)), (unsigned)z.n);
  cfg.blockDim = dim3(kFewThreads, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
#define DTB_FEW_DOWN(L)                                                                                              \
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, moe_few_down_kernel<I, G, L>, (const float*)h, w2, b2, idx, gates, y, E, H, Co, k))
  if (l2 == 16) DTB_FEW_DOWN(16);
  else if (l2 == 8) DTB_FEW_DOWN(8);
  else DTB_FEW_DOWN(4);
#undef DTB_FEW_DOWN
  count_launch(2);
}

static void moe_few(const at::Tensor& x, const at::Tensor& w1, const bf16* b1, const at::Tensor& w2, const bf16* b2,
                    const at::Tensor& idx, const at::Tensor& gates, const at::Tensor& y, const MoeSizes& z,
                    cudaStream_t st) {
  const int C = (int)w1.size(1), H = (int)w1.size(2), Co = (int)w2.size(2);
  auto h = at::empty({z.P, H}, x.options().dtype(at::kFloat));
  const auto go = [&](auto* i, auto* g) {
    moe_few_launch(bptr(x), bptr(w1), b1, bptr(w2), b2, i, g, h.data_ptr<float>(), bptr_mut(y), C, H, Co, z, st);
  };
  const bool i32 = idx.scalar_type() == at::kInt, f32 = gates.scalar_type() == at::kFloat;
  const int* pi = i32 ? idx.const_data_ptr<int>() : nullptr;
  const long* pl = i32 ? nullptr : reinterpret_cast<const long*>(idx.const_data_ptr<int64_t>());
  if (i32 && f32) go(pi, gates.const_data_ptr<float>());
  else if (i32) go(pi, bptr(gates));
  else if (f32) go(pl, gates.const_data_ptr<float>());
  else go(pl, bptr(gates));
}

template <int S>
static void launch_thin_of(const CUtensorMap& tw, const CUtensorMap& tx, const MoeThinArgs& a, long grid, cudaStream_t st) {
  static bool attr_set = false;
  if (!attr_set) {
    cudaFuncSetAttribute(moe_thin_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, MoeThinCfg<S>::SMEM_BYTES);
    attr_set = true;
  }
  launch_pdl(moe_thin_kernel<S>, dim3((unsigned)grid), kThinThreads, MoeThinCfg<S>::SMEM_BYTES, st, tw, tx, a);
}
// Four stages (two CTAs an SM), or three (three CTAs) where there are more CTAs than those hold.  In a CUDA graph with
// cold weights, two a token of 8 experts 1024 x 4096, 48 / 128 / 256 tokens: 38.8 / 39.7 / 54.3 us with four,
// 39.4 / 41.9 / 43.9 with three; four a token of 64 experts 768 x 1536, 64 tokens: 72.5 and 64.9.
static void launch_thin(const CUtensorMap& tw, const CUtensorMap& tx, const MoeThinArgs& a, const MoeSizes& z, cudaStream_t st) {
  const long each = (long)((a.N + 127) / 128) * a.splits, grid = z.R / kRowPad * each;
  const long likely = (std::min(z.P, z.E) + z.P / kRowPad) * each;  // tiles: one an expert, and the rows past them
  if (likely > 3L * num_sms()) launch_thin_of<3>(tw, tx, a, grid, st);
  else launch_thin_of<4>(tw, tx, a, grid, st);
}

// Few rows an expert, without a gradient: the plan is built, `rows` holds xp [R, C] and act [R, H].
static void moe_thin(const at::Tensor& x, const at::Tensor& w1, const bf16* b1, const at::Tensor& w2, const bf16* b2,
                     const at::Tensor& idx, const at::Tensor& gates, const at::Tensor& y, const MoePlan& pl,
                     const MoeSizes& z, cudaStream_t st) {
  const int C = (int)w1.size(1), H = (int)w1.size(2), Co = (int)w2.size(2), E = (int)z.E;
  // K is split until there are two CTAs an SM (as many tiles as experts that can have a row), 256 of K a part at least
  const long busy = std::min(z.P, z.E) * ((Co + 127) / 128);
  const int splits = (int)std::max<long>(1, std::min<long>({296 / busy, (H + 255) / 256, 16}));
  auto rows = at::empty({z.R * (C + H)}, x.options());
  auto part = at::empty({splits * z.R * Co}, x.options().dtype(at::kFloat));
  bf16 *xp = bptr_mut(rows), *act = xp + z.R * C;
  launch_pdl(moe_gather_kernel, dim3(warp_grid(z.R)), 256, 0, st, bptr(x), xp, pl, E, C, (int)z.k);
  MoeThinArgs a{pl.tile3, pl.off, E, H, C, 1, b1, act, nullptr, z.R};
  launch_thin(make_map3(bptr(w1), z.E, C, H, 64, 64), make_map(xp, z.R, C, C, 64, kRowPad), a, z, st);
  a = MoeThinArgs{pl.tile3, pl.off, E, Co, H, splits, nullptr, nullptr, part.data_ptr<float>(), z.R};
  launch_thin(make_map3(bptr(w2), z.E, H, Co, 64, 64), make_map(act, z.R, H, H, 64, kRowPad), a, z, st);
  const auto go = [&](auto* i, auto* g) {
    using I = std::remove_const_t<std::remove_pointer_t<decltype(i)>>;
    using G = std::remove_const_t<std::remove_pointer_t<decltype(g)>>;
    launch_pdl(moe_thin_combine_kernel<I, G>, dim3((unsigned)z.n, (unsigned)((Co + 511) / 512)), 128, 0, st,
               part.data_ptr<float>(), b2, i, g, bptr_mut(y), pl, E, Co, (int)z.k, splits, z.R);
  };
  const bool i32 = idx.scalar_type() == at::kInt, f32 = gates.scalar_type() == at::kFloat;
  const int* pi = i32 ? idx.const_data_ptr<int>() : nullptr;
  const long* pj = i32 ? nullptr : reinterpret_cast<const long*>(idx.const_data_ptr<int64_t>());
  if (i32 && f32) go(pi, gates.const_data_ptr<float>());
  else if (i32) go(pi, bptr(gates));
  else if (f32) go(pj, gates.const_data_ptr<float>());
  else go(pj, bptr(gates));
}

// Forward.  Returns [y] or, with `save`, [y, plan, rows] for experts_bwd.
std::vector<at::Tensor> experts_fwd(at::Tensor x, at::Tensor w1, std::optional<at::Tensor> b1, at::Tensor w2,
                                    std::optional<at::Tensor> b2, at::Tensor idx, at::Tensor gates, bool save) {
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
    return {y, none, none};
  }
  if (!save && z.P <= kFewSlots && C <= 8192) {  // x's row in shared memory
    moe_few(x, w1, bptr_opt(b1), w2, bptr_opt(b2), idx, gates, y, z, st);
    return {y};
  }
  auto plan = at::empty({plan_ints(z.P, z.E)}, x.options().dtype(at::kInt));
  const MoePlan pl = plan_views(plan.data_ptr<int>(), z.P, z.E);
  moe_build_plan(idx, pl, z, st);
  if (!save && z.P <= kThinRows * z.E) {
    moe_thin(x, w1, bptr_opt(b1), w2, bptr_opt(b2), idx, gates, y, pl, z, st);
    return {y};
  }
  // what the backward reads: the tokens' rows, the activations times their rows' gates, and the pre-activations
  auto rows = at::empty({z.R * (C + H * (save ? 2 : 1))}, x.options());
  auto yp = at::empty({z.R * Co}, x.options());
  bf16 *xp = bptr_mut(rows), *act = xp + z.R * C;
  launch_pdl(moe_gather_kernel, dim3(warp_grid(z.R)), 256, 0, st, bptr(x), xp, pl, (int)z.E, (int)C, (int)z.k);
  MoeExtra up, down;
  up.epi = MOE_GELU;
  up.bias = bptr_opt(b1);
  up.aux = save ? act + z.R * H : nullptr;
  up.gates = &gates;
  down.bias = bptr_opt(b2);
  down.gates = down.bias ? &gates : nullptr;
  moe_rows_gemm(MOE_FWD, xp, bptr(w1), act, (int)H, (int)C, up, pl, z, st);
  moe_rows_gemm(MOE_FWD, act, bptr(w2), bptr_mut(yp), (int)Co, (int)H, down, pl, z, st);
  launch_pdl(moe_combine_kernel<float>, dim3(warp_grid(z.n)), 256, 0, st, bptr(yp), bptr_mut(y), nullptr, GateParts{}, pl,
             (int)z.n, (int)Co, (int)z.k);
  if (!save) return {y};
  return {y, plan, rows};
}

// Backward: returns [dx, dgates]; the weights' and biases' gradients are written to dw1, db1, dw2, db2
// (all bf16 or all fp32; db1 / db2 only where the layer has the bias).
std::vector<at::Tensor> experts_bwd(at::Tensor dy, at::Tensor x, at::Tensor w1, at::Tensor w2, std::optional<at::Tensor> b2,
                                    at::Tensor gates, std::vector<at::Tensor> saved, at::Tensor dw1,
                                    std::optional<at::Tensor> db1, at::Tensor dw2, std::optional<at::Tensor> db2) {
  const MoeSizes z = check_experts(x, w1, std::nullopt, w2, b2, gates);
  const long C = w1.size(1), H = w1.size(2), Co = w2.size(2);
  check_bf16(dy, x, "dy");
  TORCH_CHECK(dy.dim() == 2 && dy.size(0) == z.n && dy.size(1) == Co, "experts_bwd: dy must be [n, co]");
  TORCH_CHECK(saved.size() == 2, "experts_bwd: the forward's plan and rows expected");
  const auto wt = dw1.scalar_type();
  TORCH_CHECK(wt == at::kFloat || wt == at::kBFloat16, "experts_bwd: fp32 or bf16 weight gradients");
  const auto check_grad = [&](const at::Tensor& t, at::IntArrayRef sizes, const char* what) {
    TORCH_CHECK(t.is_cuda() && t.get_device() == x.get_device() && t.scalar_type() == wt && t.sizes() == sizes &&
                    t.is_contiguous() && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0,
                "experts_bwd: ", what, " must be a contiguous, 16-byte aligned ", wt, " tensor of its weight's shape");
  };
  const bool has1 = db1 && db1->defined(), has2 = db2 && db2->defined();
  TORCH_CHECK(has2 == (bptr_opt(b2) != nullptr), "experts_bwd: b2 and db2 go together");
  check_grad(dw1, w1.sizes(), "dw1");
  check_grad(dw2, w2.sizes(), "dw2");
  if (has1) check_grad(*db1, {z.E, H}, "db1");
  if (has2) check_grad(*db2, {z.E, Co}, "db2");
  c10::cuda::CUDAGuard guard(x.device());
  bind_device_context(x.get_device());
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  auto dx = at::empty({z.n, C}, x.options());
  auto dgates = at::empty_like(gates);
  if (z.n == 0) {
    dw1.zero_();
    dw2.zero_();
    if (has1) db1->zero_();
    if (has2) db2->zero_();
    return {dx, dgates};
  }
  const at::Tensor &plan = saved[0], &rows = saved[1];
  TORCH_CHECK(plan.scalar_type() == at::kInt && plan.numel() == plan_ints(z.P, z.E) &&
                  rows.scalar_type() == at::kBFloat16 && rows.numel() == z.R * (C + 2 * H),
              "experts_bwd: saved tensors of another forward");
  const MoePlan pl = plan_views(plan.data_ptr<int>(), z.P, z.E);
  const bf16 *xp = bptr(rows), *act = xp + z.R * C;
  bf16* pre = bptr_mut(rows) + z.R * (C + H);
  // scratch: dpre, dy's rows (later dx's); fp32: the rows' products, the column sums of blocks of rows
  const int parts = moe_dot_parts((int)H, z);
  const int bparts = has2 ? (int)((Co + 255) / 256) : 0;
  const long sums = has1 ? z.R / 32 * H : 0, sums2 = has2 ? z.R / kRowPad * Co : 0;
  const long wide = std::max(C, Co);
  auto scratch = at::empty({z.R * (H + wide) + 2 * (z.R * (parts + bparts) + sums + sums2)}, x.options());
  bf16* dpre = bptr_mut(scratch);
  bf16* dyp = dpre + z.R * H;
  bf16* dxp = dyp;
  float* dots = reinterpret_cast<float*>(dyp + z.R * wide);
  float* bias_dots = has2 ? dots + z.R * parts : nullptr;
  float* p1 = has1 ? dots + z.R * (parts + bparts) : nullptr;
  float* p2 = has2 ? dots + z.R * (parts + bparts) + sums : nullptr;
  const auto dy_rows = [&](auto* g) {
    using G = std::remove_const_t<std::remove_pointer_t<decltype(g)>>;
    const dim3 grid((unsigned)std::min<long>(z.R / kRowPad, 1L << 16), (unsigned)((Co + 255) / 256));
    moe_dy_rows_kernel<G><<<grid, 256, 0, st>>>(bptr(dy), bptr_opt(b2), g, dyp, p2, bias_dots, pl, (int)z.E, (int)Co,
                                                (int)z.k, z.R);
  };
  if (gates.scalar_type() == at::kFloat) dy_rows(gates.const_data_ptr<float>());
  else dy_rows(bptr(gates));
  count_launch();
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  MoeExtra back;
  back.epi = MOE_DGELU;
  back.aux = pre;
  back.sums = p1;
  back.dots = dots;
  back.gates = &gates;
  moe_rows_gemm(MOE_DX, dyp, bptr(w2), dpre, (int)H, (int)Co, back, pl, z, st);
  moe_weight_gemm(act, dyp, dw2, (int)H, (int)Co, pl, z, st);
  moe_rows_gemm(MOE_DX, dpre, bptr(w1), dxp, (int)C, (int)H, MoeExtra{}, pl, z, st);
  moe_weight_gemm(xp, dpre, dw1, (int)C, (int)H, pl, z, st);
  if (has1 || has2) {
    const auto join = [&](auto* o1, auto* o2) {
      using O = std::remove_pointer_t<decltype(o1)>;
      JoinArgs<O> a{p1, o1, (int)H, 32}, b{p2, o2, (int)Co, kRowPad};
      const long widest = std::max(has1 ? H : 0, has2 ? Co : 0);
      const dim3 grid((unsigned)((widest + 63) / 64), (unsigned)z.E, has1 && has2 ? 2 : 1);
      launch_pdl(moe_join_sums_kernel<O>, grid, 256, 0, st, has1 ? a : b, b, pl);
    };
    if (wt == at::kFloat) join(has1 ? db1->data_ptr<float>() : nullptr, has2 ? db2->data_ptr<float>() : nullptr);
    else join(has1 ? bptr_mut(*db1) : nullptr, has2 ? bptr_mut(*db2) : nullptr);
  }
  const GateParts gp{dots, bias_dots, parts, bparts, z.R};
  const auto last = [&](auto* dg) {
    using G = std::remove_pointer_t<decltype(dg)>;
    launch_pdl(moe_combine_kernel<G>, dim3(warp_grid(z.n)), 256, 0, st, (const bf16*)dxp, bptr_mut(dx), dg, gp, pl, (int)z.n,
               (int)C, (int)z.k);
  };
  if (gates.scalar_type() == at::kFloat) last(dgates.data_ptr<float>());
  else last(bptr_mut(dgates));
  return {dx, dgates};
}

DTB_DEFINE_STATUS_READER(status_moe)

}  // namespace dtb
