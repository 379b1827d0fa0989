// Routing of tokens to experts: scores, choice of k experts a token, gates, and the
// gates' gradient with respect to the logits.  (No counterpart in the reference,
// whose MLPs are dense: dtrain/nn.py:90-101.)
//
//   s = softmax(z) or 1 / (1 + exp(-z))          z = logits, fp32; -inf masks an expert
//   c = z, or s + bias with a balancing bias     what the choice goes by
//   groups: the keep best of G equal groups stay, by their best c or their two best
//   idx = the k largest c (ties: lowest expert), gates = scale * s[idx] / max(sum, 1e-20)
//
// Both scores increase with z, so without a bias the choice goes by the logits
// themselves: no two experts are made equal by rounding their scores.  A NaN counts as
// the largest value, so it is chosen and shows in the gates.  Slots that no expert is
// left for (a row of masked experts) get idx -1 and gate 0.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAException.h>

#include "common.cuh"

namespace dtb {

constexpr int kRouteMaxExperts = 512;
constexpr int kRouteMaxK = 32;
constexpr float kRouteTiny = 1e-20f;  // the renormalising sum is at least this
constexpr unsigned kAll = 0xffffffffu;

struct RouteArgs {
  const void* logits;
  const float* bias;
  float* gates;
  int* idx;
  int* load;
  int n, e, k;
  int groups, keep, top;
  int softmax, renorm;
  int log_lanes; // route_fwd_kernel: log2 of a group's lanes
  int vec;       // its lanes' values start at 16-byte boundaries
  int need_sum;  // the softmax's sum takes part: not when the gates are renormalised over the row's largest
  float scale;
};

// Unsigned keys in the order of the floats, -0 = +0, NaN above +inf; 0 is free for
// "taken or absent" (the key of -inf is above it).
__device__ __forceinline__ unsigned order_key(float x) {
  if (x != x) return 0xffffffffu;
  const int b = __float_as_int(x + 0.f);
  return (unsigned)(b ^ ((b >> 31) | (int)0x80000000));
}
constexpr unsigned kKeyNegInf = 0x007fffffu;
__device__ __forceinline__ float key_value(unsigned k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

__device__ __forceinline__ float load_logit(const float* p) { return *p; }
__device__ __forceinline__ float load_logit(const bf16* p) { return bf2f(*p); }
__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_logit(bf16* p, float v) { *p = f2bf(v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
__device__ __forceinline__ float sigmoid_f(float z) { return __frcp_rn(1.f + expf(-z)); }

// The gates of the chosen experts (lane j: slot j).
template <typename T>
__device__ __forceinline__ void route_finish(const RouteArgs& a, const T* row, int t, int lane, int mine, float mx,
                                             float sum, int* s_load) {
  float sj = 0.f;
  if (mine >= 0) {
    const float zj = load_logit(row + mine);
    sj = a.softmax ? expf(zj - mx) / sum : sigmoid_f(zj);
    atomicAdd(&s_load[mine], 1);
  }
  float d = 1.f;
  if (a.renorm) {
    const float total = warp_sum(sj);
    d = total < kRouteTiny ? kRouteTiny : total;
  }
  if (lane < a.k) {
    a.gates[(long)t * a.k + lane] = mine >= 0 ? a.scale * sj / d : 0.f;
    a.idx[(long)t * a.k + lane] = mine;
  }
}
__device__ __forceinline__ void route_counts(const RouteArgs& a, const int* s_load) {
  __syncthreads();
  for (int i = threadIdx.x; i < a.e; i += blockDim.x) {
    if (gridDim.x == 1) a.load[i] = s_load[i];
    else if (s_load[i]) atomicAdd(a.load + i, s_load[i]);
  }
}

// V values of a row from `p` on, of which the first `valid` are there (vec: all, 16-byte aligned).
template <typename T, int V>
__device__ __forceinline__ void load_logits(const T* p, int valid, bool vec, float* z) {
  constexpr int PER16 = 16 / (int)sizeof(T);
  if constexpr (V % PER16 == 0) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < V / PER16; ++i) {
        const uint4 u = *(reinterpret_cast<const uint4*>(p) + i);  // p: global or shared memory
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (sizeof(T) == 4) {
            z[i * 4 + j] = __uint_as_float(w[j]);
          } else {
            z[i * 8 + 2 * j] = __uint_as_float(w[j] << 16);
            z[i * 8 + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
          }
        }
      }
      return;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) z[v] = v < valid ? load_logit(p + v) : -INFINITY;
}
template <typename T, int V>
__device__ __forceinline__ void store_logits(T* p, int valid, bool vec, const float* z) {
  constexpr int PER16 = 16 / (int)sizeof(T);
  if constexpr (V % PER16 == 0) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < V / PER16; ++i) {
        uint4 u;
        if constexpr (sizeof(T) == 4)
          u = make_uint4(__float_as_uint(z[4 * i]), __float_as_uint(z[4 * i + 1]), __float_as_uint(z[4 * i + 2]),
                         __float_as_uint(z[4 * i + 3]));
        else
          u = make_uint4(pack_bf16x2(z[8 * i], z[8 * i + 1]), pack_bf16x2(z[8 * i + 2], z[8 * i + 3]),
                         pack_bf16x2(z[8 * i + 4], z[8 * i + 5]), pack_bf16x2(z[8 * i + 6], z[8 * i + 7]));
        *(reinterpret_cast<uint4*>(p) + i) = u;
      }
      return;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (v < valid) store_logit(p + v, z[v]);
}

// One warp per token.  The lanes are split evenly over the groups (their number rounded up
// to a power of two), and each lane holds V experts in a row of its group, sorted once by
// a stable exchange of neighbours; lanes stand in the experts' order, so the lowest lane
// that holds a largest key holds the lowest such expert.  A group's two best come from the
// heads of its lanes' lists by xor-shuffles, all groups at once, and each of the k rounds
// takes the largest head of the warp (redux) and pops it.
//
// Bound by instruction issue, most of it integer work (scores, keys, the sort, the pops): 1055 instructions a
// token at 256 experts in 8 groups, 8 a token (issue 71% of the active cycles, the half-rate integer pipe 54% of
// all).  65536 such tokens, fp32: 82 us (71 MB, 11 us at the copy rate).  The experts of groups that are dropped
// are sorted too, since that comes first.  Unsorted values rescanned each round (route_fwd_wide_kernel) took
// 194 us there; that form serves V > 8, where the sort would cost more.
template <typename T, int V>
__global__ void __launch_bounds__(256) route_fwd_kernel(RouteArgs a) {
  extern __shared__ int s_load[];
  for (int i = threadIdx.x; i < a.e; i += blockDim.x) s_load[i] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int warps = (gridDim.x * blockDim.x) >> 5;
  const int per = a.e / a.groups;
  const int lanes = 1 << a.log_lanes;  // of a group
  const int group = lane >> a.log_lanes, part = lane & (lanes - 1);
  const int base = group * per + part * V;
  const int valid = group < a.groups ? max(0, min(V, per - part * V)) : 0;
  const bool by_score = a.bias != nullptr || a.top == 2;
  float bias[V];
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = a.bias != nullptr && v < valid ? a.bias[base + v] : 0.f;
  for (int t = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; t < a.n; t += warps) {
    const T* row = reinterpret_cast<const T*>(a.logits) + (long)t * a.e;
    float z[V];
    load_logits<T, V>(row + base, valid, a.vec && valid == V, z);
    float mx = 0.f, sum = 1.f;  // softmax: s = exp(z - mx) / sum
    if (a.softmax) {
      float m = z[0];
#pragma unroll
      for (int v = 1; v < V; ++v) m = fmaxf(m, z[v]);
      m = warp_max(m);
      mx = m == -INFINITY ? 0.f : m;
      if (a.need_sum) {
        float p = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) p += expf(z[v] - mx);
        sum = warp_sum(p);
        if (sum == 0.f) sum = 1.f;
      }
    }
    unsigned key[V];
    int at[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float c = z[v];
      if (by_score) {
        c = a.softmax ? expf(z[v] - mx) / sum : sigmoid_f(z[v]);
        if (a.bias != nullptr) c = __fadd_rn(c, bias[v]);
        if (z[v] == -INFINITY) c = -INFINITY;
      }
      key[v] = order_key(c);  // absent experts: -inf, as masked ones
      at[v] = v;
    }
#pragma unroll
    for (int i = 0; i < V - 1; ++i)
#pragma unroll
      for (int j = 0; j < V - 1 - i; ++j)
        if (key[j + 1] > key[j]) {
          const unsigned k0 = key[j];
          const int a0 = at[j];
          key[j] = key[j + 1];
          at[j] = at[j + 1];
          key[j + 1] = k0;
          at[j + 1] = a0;
        }
    unsigned where = 0u;  // the list's experts, four bits each
#pragma unroll
    for (int v = 0; v < V; ++v) where |= (unsigned)at[v] << (4 * v);
    if (a.groups > 1) {
      unsigned k1 = key[0], k2 = 0u;
      if constexpr (V > 1) k2 = key[1];
      for (int o = 1; o < lanes; o <<= 1) {
        const unsigned b1 = __shfl_xor_sync(kAll, k1, o), b2 = __shfl_xor_sync(kAll, k2, o);
        k2 = max(min(k1, b1), max(k2, b2));
        k1 = max(k1, b1);
      }
      unsigned score = k1;
      if (a.top == 2 && k1 > kKeyNegInf && k2 > kKeyNegInf)
        score = order_key(__fadd_rn(key_value(k1), key_value(k2)));
      // the group's place among the groups: those with a larger score, or an equal one and a lower number
      int place = 0;
      for (int g = 0; g < a.groups; ++g) {
        const unsigned other = __shfl_sync(kAll, score, g << a.log_lanes);
        place += other > score || (other == score && g < group);
      }
      if (place >= a.keep) {
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = 0u;
      }
    }
    int mine = -1;
    for (int j = 0; j < a.k; ++j) {
      const unsigned best = __reduce_max_sync(kAll, key[0]);
      if (best <= kKeyNegInf) break;
      const int l = __ffs(__ballot_sync(kAll, key[0] == best)) - 1;
      const int i = __shfl_sync(kAll, base + (int)(where & 15u), l);
      if (lane == j) mine = i;
      const bool pop = lane == l;
#pragma unroll
      for (int v = 0; v < V - 1; ++v) key[v] = pop ? key[v + 1] : key[v];
      key[V - 1] = pop ? 0u : key[V - 1];
      where = pop ? where >> 4 : where;
    }
    route_finish(a, row, t, lane, mine, mx, sum, s_load);
  }
  route_counts(a, s_load);
}

// One warp per token; lane l holds experts l, l + 32, ... unsorted: any groups and sizes.
template <typename T, int VPL>
__global__ void __launch_bounds__(256) route_fwd_wide_kernel(RouteArgs a) {
  extern __shared__ int s_load[];
  for (int i = threadIdx.x; i < a.e; i += blockDim.x) s_load[i] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int warps = (gridDim.x * blockDim.x) >> 5;
  const int per = a.e / a.groups;
  for (int t = (blockIdx.x * blockDim.x + threadIdx.x) >> 5; t < a.n; t += warps) {
    const T* row = reinterpret_cast<const T*>(a.logits) + (long)t * a.e;
    float z[VPL];
    unsigned key[VPL];
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const int i = v * 32 + lane;
      z[v] = i < a.e ? load_logit(row + i) : -INFINITY;
      m = fmaxf(m, z[v]);
    }
    float mx = 0.f, sum = 1.f;  // softmax: s = exp(z - mx) / sum
    if (a.softmax) {
      m = warp_max(m);
      mx = m == -INFINITY ? 0.f : m;
      float p = 0.f;
#pragma unroll
      for (int v = 0; v < VPL; ++v) p += expf(z[v] - mx);
      sum = warp_sum(p);
      if (sum == 0.f) sum = 1.f;
    }
    const bool by_score = a.bias != nullptr || a.top == 2;
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      const int i = v * 32 + lane;
      float c = z[v];
      if (by_score && z[v] != -INFINITY) {
        c = a.softmax ? expf(z[v] - mx) / sum : sigmoid_f(z[v]);
        if (a.bias) c = __fadd_rn(c, a.bias[i]);
      }
      key[v] = i < a.e ? order_key(c) : 0u;
    }
    if (a.groups > 1) {
      // lane g keeps the score of group g
      unsigned gk = 0u;
      for (int g = 0; g < a.groups; ++g) {
        unsigned k1 = 0u, k2 = 0u;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
          const int i = v * 32 + lane;
          const unsigned k = (i >= g * per && i < (g + 1) * per) ? key[v] : 0u;
          k2 = max(k2, min(k1, k));
          k1 = max(k1, k);
        }
        const unsigned best = __reduce_max_sync(kAll, k1);
        unsigned sc = best;
        if (a.top == 2) {
          const int first = __ffs(__ballot_sync(kAll, k1 == best)) - 1;
          const unsigned second = __reduce_max_sync(kAll, lane == first ? k2 : k1);
          if (best > kKeyNegInf && second > kKeyNegInf)
            sc = order_key(__fadd_rn(key_value(best), key_value(second)));
        }
        if (lane == g) gk = sc;
      }
      unsigned kept = 0u;
      for (int r = 0; r < a.keep; ++r) {
        const unsigned best = __reduce_max_sync(kAll, gk);
        const int g = __ffs(__ballot_sync(kAll, gk == best)) - 1;
        kept |= 1u << g;
        if (lane == g) gk = 0u;
      }
#pragma unroll
      for (int v = 0; v < VPL; ++v) {
        const int i = v * 32 + lane;
        if (i < a.e && !((kept >> (i / per)) & 1u)) key[v] = 0u;
      }
    }
    // k rounds: the largest key, ties to the lowest expert
    int mine = -1;
    unsigned lk = 0u;
    int lv = 0;
#pragma unroll
    for (int v = VPL - 1; v >= 0; --v)
      if (key[v] >= lk) { lk = key[v]; lv = v; }
    for (int j = 0; j < a.k; ++j) {
      const unsigned best = __reduce_max_sync(kAll, lk);
      if (best <= kKeyNegInf) break;
      const int i = __reduce_min_sync(kAll, lk == best ? lv * 32 + lane : 0x7fffffff);
      if (lane == j) mine = i;
      if ((i & 31) == lane) {
        lk = 0u;
#pragma unroll
        for (int v = VPL - 1; v >= 0; --v) {
          if (v == (i >> 5)) key[v] = 0u;
          if (key[v] >= lk) { lk = key[v]; lv = v; }
        }
      }
    }
    route_finish(a, row, t, lane, mine, mx, sum, s_load);
  }
  route_counts(a, s_load);
}

struct RouteBwdArgs {
  const void* logits;
  const int* idx;
  const float* dgates;
  void* dlogits;
  int n, e, k;
  int softmax, renorm;
  int vec;  // the lanes' values start at 16-byte boundaries
  float scale;
};

// One warp per token.  With D = max(S, tiny), S the sum of the chosen s:
//   ds_j = scale / D (G_j - [renorm, S > tiny] sum_i G_i s_i / D)
//   sigmoid: dz_j = ds_j s_j (1 - s_j);  softmax: dz_i = s_i (ds_i - sum_j ds_j s_j)
// The row is put together in shared memory (each lane owns V experts in a row) and
// written with 16-byte stores.  The sigmoid reads the chosen logits only, the softmax the
// row; both write the row.  Bound by the latency of the chain choice, logit, row: 65536 x 256
// fp32, 8 a token, sigmoid, takes 23 us (71 MB, 3.1 TB/s).
template <typename T, int V>
__global__ void __launch_bounds__(256) route_bwd_kernel(RouteBwdArgs a) {
  extern __shared__ __align__(16) float s_row[];
  const int lane = threadIdx.x & 31;
  const int warps = (gridDim.x * blockDim.x) >> 5;
  float* buf = s_row + (threadIdx.x >> 5) * (32 * V);
  const int base = lane * V;
  const int valid = max(0, min(V, a.e - base));
  const bool vec = a.vec && valid == V;
  int t = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  // the next token's choices are loaded while this one is worked on
  int next_at = -1;
  float next_G = 0.f;
  const auto fetch = [&](int n) {
    next_at = -1;
    if (n < a.n && lane < a.k) {
      next_at = a.idx[(long)n * a.k + lane];
      next_G = a.dgates[(long)n * a.k + lane];
    }
  };
  fetch(t);
  for (; t < a.n; t += warps) {
    const T* row = reinterpret_cast<const T*>(a.logits) + (long)t * a.e;
    T* out = reinterpret_cast<T*>(a.dlogits) + (long)t * a.e;
    int at = next_at < a.e ? next_at : -1;
    if (at < 0) at = -1;
    const float G = at >= 0 ? next_G : 0.f;
    const float zj = at >= 0 ? load_logit(row + at) : 0.f;
    fetch(t + warps);
    float w[V];
#pragma unroll
    for (int v = 0; v < V; ++v) w[v] = 0.f;
    store_logits<float, V>(buf + base, V, true, w);
    float m = 0.f, sum = 1.f;
    if (a.softmax) {
      load_logits<T, V>(row + base, valid, vec, w);
      m = w[0];
#pragma unroll
      for (int v = 1; v < V; ++v) m = fmaxf(m, w[v]);
      m = warp_max(m);
      if (m == -INFINITY) m = 0.f;
      float p = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        w[v] = expf(w[v] - m);
        p += w[v];
      }
      sum = warp_sum(p);
      if (sum == 0.f) sum = 1.f;
    }
    float s = 0.f;
    if (at >= 0) s = a.softmax ? expf(zj - m) / sum : sigmoid_f(zj);
    float ds = G;
    if (a.renorm) {
      const float total = warp_sum(s);
      const float d = total < kRouteTiny ? kRouteTiny : total;
      const float dot = warp_sum(G * s) / d;
      ds = (G - (total > kRouteTiny ? dot : 0.f)) / d;
    }
    ds = at >= 0 ? a.scale * ds : 0.f;
    const float back = a.softmax ? warp_sum(ds * s) : 0.f;
    __syncwarp();
    if (at >= 0) buf[at] = a.softmax ? ds : ds * s * (1.f - s);
    __syncwarp();
    float b[V];
    load_logits<float, V>(buf + base, V, true, b);
    if (a.softmax) {
#pragma unroll
      for (int v = 0; v < V; ++v) b[v] = w[v] / sum * (b[v] - back);
    }
    store_logits<T, V>(out + base, valid, vec, b);
    __syncwarp();
  }
}

// Eight warps a CTA, one token each at a time.
static int route_grid(int n) { return (int)std::max<long>(1, std::min<long>((n + 7) / 8, 148L * 8)); }

// Logits [n, e] (fp32 or bf16, contiguous) -> gates fp32 [n, k], idx int32 [n, k], load int32 [e].
std::vector<at::Tensor> route_fwd(at::Tensor logits, int64_t k, bool softmax, std::optional<at::Tensor> bias,
                                     int64_t groups, int64_t keep, int64_t top, bool renorm, double scale) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.is_contiguous(), "route: contiguous [n, e] CUDA logits");
  const bool f32 = logits.scalar_type() == at::kFloat;
  TORCH_CHECK(f32 || logits.scalar_type() == at::kBFloat16, "route: fp32 or bf16 logits");
  const long n = logits.size(0), e = logits.size(1);
  TORCH_CHECK(e >= 1 && e <= kRouteMaxExperts, "route: 1 to ", kRouteMaxExperts, " experts, got ", e);
  TORCH_CHECK(k >= 1 && k <= e && k <= kRouteMaxK, "route: k must be in [1, min(experts, ", kRouteMaxK, ")], got ", k);
  TORCH_CHECK(n < (1L << 31) / 32, "route: too many rows");
  TORCH_CHECK(groups >= 1 && groups <= 32 && e % groups == 0, "route: groups must divide the experts, at most 32");
  TORCH_CHECK(keep >= 1 && keep <= groups && keep * (e / groups) >= k, "route: the kept groups hold fewer than k experts");
  TORCH_CHECK(top == 1 || (top == 2 && e / groups >= 2), "route: group_top must be 1, or 2 with groups of at least 2");
  c10::cuda::CUDAGuard guard(logits.device());
  RouteArgs a{};
  if (bias && bias->defined()) {
    TORCH_CHECK(bias->is_cuda() && bias->get_device() == logits.get_device() && bias->scalar_type() == at::kFloat &&
                    bias->numel() == e && bias->is_contiguous(),
                "route: bias must be fp32 [experts] on the logits' device");
    a.bias = bias->data_ptr<float>();
  }
  auto gates = at::empty({n, k}, logits.options().dtype(at::kFloat));
  auto idx = at::empty({n, k}, logits.options().dtype(at::kInt));
  auto load = at::empty({e}, logits.options().dtype(at::kInt));
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  const int grid = route_grid((int)n);
  if (grid > 1 || n == 0) C10_CUDA_CHECK(cudaMemsetAsync(load.data_ptr(), 0, e * 4, st));  // one CTA writes its counts
  if (n == 0) return {gates, idx, load};
  a.logits = logits.data_ptr();
  a.gates = gates.data_ptr<float>();
  a.idx = idx.data_ptr<int>();
  a.load = load.data_ptr<int>();
  a.n = (int)n;
  a.e = (int)e;
  a.k = (int)k;
  a.groups = (int)groups;
  a.keep = (int)keep;
  a.top = (int)top;
  a.softmax = softmax;
  a.renorm = renorm;
  a.scale = (float)scale;
  a.need_sum = !(renorm && !a.bias && groups == 1 && top == 1);
  a.log_lanes = 5;
  while ((32 >> a.log_lanes) < groups) --a.log_lanes;
  const long per = e / groups, lanes = 1 << a.log_lanes, v = (per + lanes - 1) / lanes;
  const int V = v <= 1 ? 1 : v <= 2 ? 2 : v <= 4 ? 4 : 8;
  const int es = f32 ? 4 : 2;
  a.vec = per % V == 0 && (V * es) % 16 == 0 && (e * es) % 16 == 0 &&
          (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0;
#define DTB_ROUTE(KERN, V)                                              \
  if (f32) KERN<float, V><<<grid, 256, e * 4, st>>>(a);                 \
  else KERN<bf16, V><<<grid, 256, e * 4, st>>>(a);
  if (v <= 1) { DTB_ROUTE(route_fwd_kernel, 1) }
  else if (v <= 2) { DTB_ROUTE(route_fwd_kernel, 2) }
  else if (v <= 4) { DTB_ROUTE(route_fwd_kernel, 4) }
  else if (v <= 8) { DTB_ROUTE(route_fwd_kernel, 8) }
  else if (e <= 256) { DTB_ROUTE(route_fwd_wide_kernel, 8) }
  else { DTB_ROUTE(route_fwd_wide_kernel, 16) }
#undef DTB_ROUTE
  count_launch();
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {gates, idx, load};
}

// d(logits) in the logits' type from the gates' gradient (fp32 [n, k]).
at::Tensor route_bwd(at::Tensor logits, at::Tensor idx, at::Tensor dgates, bool softmax, bool renorm, double scale) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.is_contiguous(), "route_bwd: contiguous CUDA logits");
  const bool f32 = logits.scalar_type() == at::kFloat;
  TORCH_CHECK(f32 || logits.scalar_type() == at::kBFloat16, "route_bwd: fp32 or bf16 logits");
  const long n = logits.size(0), e = logits.size(1);
  TORCH_CHECK(idx.dim() == 2 && idx.size(0) == n && idx.scalar_type() == at::kInt && idx.is_contiguous(), "route_bwd: idx");
  const long k = idx.size(1);
  TORCH_CHECK(e <= kRouteMaxExperts && k >= 1 && k <= kRouteMaxK && k <= e, "route_bwd: sizes");
  TORCH_CHECK(dgates.sizes() == idx.sizes() && dgates.scalar_type() == at::kFloat && dgates.is_contiguous() &&
                  dgates.device() == logits.device() && idx.device() == logits.device(),
              "route_bwd: dgates");
  c10::cuda::CUDAGuard guard(logits.device());
  auto dl = at::empty_like(logits);
  if (n == 0) return dl;
  RouteBwdArgs a{logits.data_ptr(), idx.data_ptr<int>(), dgates.data_ptr<float>(), dl.data_ptr(), (int)n, (int)e, (int)k, softmax, renorm, 0, (float)scale};
  const int V = e <= 32 ? 1 : e <= 64 ? 2 : e <= 128 ? 4 : e <= 256 ? 8 : 16;
  const int es = f32 ? 4 : 2;
  a.vec = (V * es) % 16 == 0 && (e * es) % 16 == 0 &&
          ((reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.dlogits)) & 15) == 0;
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  const int grid = route_grid(a.n);
#define DTB_ROUTE(V)                                                             \
  if (f32) route_bwd_kernel<float, V><<<grid, 256, 8 * 32 * V * 4, st>>>(a);     \
  else route_bwd_kernel<bf16, V><<<grid, 256, 8 * 32 * V * 4, st>>>(a);
  if (V == 1) { DTB_ROUTE(1) }
  else if (V == 2) { DTB_ROUTE(2) }
  else if (V == 4) { DTB_ROUTE(4) }
  else if (V == 8) { DTB_ROUTE(8) }
  else { DTB_ROUTE(16) }
#undef DTB_ROUTE
  count_launch();
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return dl;
}

}  // namespace dtb
