// Global gradient norm over many tensors, and clipping, in two launches.
//
//   norm = sqrt(sum over tensors and elements of g^2)
//   f = 1 if norm <= max_norm (or norm is 0), else max_norm / (norm + 1e-6)
//   out = g * f                       in place, or into tensors of another type
//
// The factor is the one of dtrain/optim.py:49-52; csrc/optim.cu applies it to one flat
// fp32 buffer, this file to a list of tensors of any sizes, types and layouts (a
// mixture of experts' parameters, bf16 gradients bound for the flat fp32 buffer).
//
// The list travels in the kernels' parameters (32 bytes a tensor, up to 960 tensors a
// launch), so there is no copy to the device and the calls can be captured in a CUDA
// graph.  Each CTA of the first kernel sums its chunks in a fixed order into one fp64
// partial; each CTA of the second adds the partials up in the same order, so every CTA
// gets the same factor, and the result does not depend on scheduling.
//
// Bound by memory: the gradients are read twice (the norm has to be known before the first of
// them is scaled) and written once.  406M fp32 gradients: norm 250 us (6.5 TB/s), scaling
// 530 us (6.1 TB/s; it starts with the chunks that the norm left in L2); 266M bf16 ones into
// fp32: 113 and 261 us.  A few small tensors: two launches, 7.5 us on the GPU.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "overlap.h"

namespace dtb {

constexpr int kClipThreads = 256;
constexpr int kClipChunk = 8192;     // elements of a tensor that a CTA takes at a time
constexpr int kClipGrid = 148 * 4;   // most CTAs of a launch: fixed, so the order of the sums is too
constexpr int kClipStridedMax = 128;

enum ClipType : int { CLIP_F32 = 0, CLIP_BF16 = 1, CLIP_F16 = 2 };

struct ClipDesc {
  const void* in;
  void* out;   // null where only the norm is asked for
  long n;
  int first;   // chunks of the tensors before this one
  short in_t, out_t;
};
template <int CAP>
struct ClipList {
  int count, chunks;
  ClipDesc d[CAP];
};
// A tensor that is not dense, or whose output has another order of its elements.
struct ClipStrided {
  const void* in;
  void* out;
  long n;
  int size[4];
  long is[4], os[4];
  short in_t, out_t;
};
struct ClipStridedList {
  int count;
  ClipStrided d[kClipStridedMax];
};

__device__ __forceinline__ float clip_load(const void* p, int t, long i) {
  if (t == CLIP_F32) return reinterpret_cast<const float*>(p)[i];
  if (t == CLIP_BF16) return bf2f(reinterpret_cast<const bf16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void clip_store(void* p, int t, long i, float v) {
  if (t == CLIP_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (t == CLIP_BF16) reinterpret_cast<bf16*>(p)[i] = f2bf(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

// The values of one 16-byte load: 4 fp32, or 8 of 16 bits.
template <int T>
struct ClipVec;
template <>
struct ClipVec<CLIP_F32> {
  static constexpr int N = 4;
  static constexpr unsigned kMask = 0x7fffffffu;
  static __device__ __forceinline__ void get(const uint4& u, float* v) {
    v[0] = __uint_as_float(u.x);
    v[1] = __uint_as_float(u.y);
    v[2] = __uint_as_float(u.z);
    v[3] = __uint_as_float(u.w);
  }
};
template <>
struct ClipVec<CLIP_BF16> {
  static constexpr int N = 8;
  static constexpr unsigned kMask = 0x7fff7fffu;
  static __device__ __forceinline__ void get(const uint4& u, float* v) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <>
struct ClipVec<CLIP_F16> {
  static constexpr int N = 8;
  static constexpr unsigned kMask = 0x7fff7fffu;
  static __device__ __forceinline__ void get(const uint4& u, float* v) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
};

// Sum of the squares of one 16-byte load: in fp32, added to an fp64 total by the caller.
// Where fp32 squares would overflow or vanish (the values are not zero), in fp64.
template <int T>
__device__ __forceinline__ double clip_squares(const uint4& u) {
  float v[ClipVec<T>::N];
  ClipVec<T>::get(u, v);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < ClipVec<T>::N; ++i) s = fmaf(v[i], v[i], s);
  if (!(s <= 1e38f) || (s < 1e-30f && ((u.x | u.y | u.z | u.w) & ClipVec<T>::kMask))) {
    double d = 0.0;
#pragma unroll
    for (int i = 0; i < ClipVec<T>::N; ++i) d += (double)v[i] * (double)v[i];
    return d;
  }
  return (double)s;
}

template <class List>
__device__ __forceinline__ int clip_find(const List& l, int chunk) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.d[mid].first <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// [lo, hi) elements of the chunk, and the head: elements before the first 16-byte boundary.
struct ClipSpan {
  long lo;
  int head, vecs, len;
};
template <int T>
__device__ __forceinline__ ClipSpan clip_span(const ClipDesc& d, int chunk) {
  constexpr int N = ClipVec<T>::N, S = 16 / N;
  ClipSpan s;
  s.lo = (long)(chunk - d.first) * kClipChunk;
  s.len = (int)min((long)kClipChunk, d.n - s.lo);
  const unsigned off = (unsigned)((reinterpret_cast<uintptr_t>(d.in) + s.lo * S) & 15);
  s.head = min(s.len, off ? (int)(16 - off) / S : 0);
  s.vecs = (s.len - s.head) / N;
  return s;
}

template <int T>
__device__ __forceinline__ double clip_chunk_squares(const ClipDesc& d, int chunk) {
  constexpr int N = ClipVec<T>::N, S = 16 / N;
  const ClipSpan s = clip_span<T>(d, chunk);
  const char* base = reinterpret_cast<const char*>(d.in) + s.lo * S;
  double acc = 0.0;
  const uint4* p = reinterpret_cast<const uint4*>(base + s.head * S);
  constexpr int U = 4;
  int i = threadIdx.x;
  for (; i + (U - 1) * kClipThreads < s.vecs; i += U * kClipThreads) {
    uint4 u[U];
#pragma unroll
    for (int j = 0; j < U; ++j) u[j] = __ldg(p + i + j * kClipThreads);
#pragma unroll
    for (int j = 0; j < U; ++j) acc += clip_squares<T>(u[j]);
  }
  for (; i < s.vecs; i += kClipThreads) acc += clip_squares<T>(__ldg(p + i));
  for (int e = threadIdx.x; e < s.len - s.vecs * N; e += kClipThreads) {
    const double x = (double)clip_load(base, T, e < s.head ? e : e + s.vecs * N);
    acc += x * x;
  }
  return acc;
}

// Sum over the CTA in a fixed order; every thread gets it.
__device__ __forceinline__ double clip_block_sum(double v) {
  __shared__ double sm[kClipThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kClipThreads / 32; ++w) s += sm[w];
  __syncthreads();
  return s;
}

template <int CAP>
__global__ void __launch_bounds__(kClipThreads)
    clip_norm_kernel(const __grid_constant__ ClipList<CAP> l, double* __restrict__ part) {
  double acc = 0.0;
  for (int c = blockIdx.x; c < l.chunks; c += gridDim.x) {
    const ClipDesc& d = l.d[clip_find(l, c)];
    if (d.in_t == CLIP_F32) acc += clip_chunk_squares<CLIP_F32>(d, c);
    else if (d.in_t == CLIP_BF16) acc += clip_chunk_squares<CLIP_BF16>(d, c);
    else acc += clip_chunk_squares<CLIP_F16>(d, c);
  }
  acc = clip_block_sum(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

__device__ __forceinline__ long clip_offset(const int* size, const long* st, long i) {
  long o = 0;
#pragma unroll
  for (int k = 3; k >= 0; --k) {
    o += (i % size[k]) * st[k];
    i /= size[k];
  }
  return o;
}

__global__ void __launch_bounds__(kClipThreads)
    clip_norm_strided_kernel(const __grid_constant__ ClipStridedList l, double* __restrict__ part) {
  double acc = 0.0;
  for (int t = 0; t < l.count; ++t) {
    const ClipStrided& d = l.d[t];
    for (long i = (long)blockIdx.x * kClipThreads + threadIdx.x; i < d.n; i += (long)gridDim.x * kClipThreads) {
      const double x = (double)clip_load(d.in, d.in_t, clip_offset(d.size, d.is, i));
      acc += x * x;
    }
  }
  acc = clip_block_sum(acc);
  if (threadIdx.x == 0) part[blockIdx.x] = acc;
}

// The factor from the partials; CTA 0 of the launch that has `norm` writes it.
__device__ __forceinline__ float clip_total(const double* part, int np, float max_norm, float* norm) {
  double s = 0.0;
  for (int i = threadIdx.x; i < np; i += kClipThreads) s += __ldcg(part + i);
  const double n = sqrt(clip_block_sum(s));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  if (n <= (double)max_norm || n == 0.0) return 1.f;
  return (float)((double)max_norm / (n + 1e-6));
}

template <int T>
__device__ __forceinline__ void clip_store_vec(void* out, long i, const float* v);
template <>
__device__ __forceinline__ void clip_store_vec<CLIP_F32>(void* out, long i, const float* v) {
  __stcs(reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + i), make_float4(v[0], v[1], v[2], v[3]));
}
template <>
__device__ __forceinline__ void clip_store_vec<CLIP_BF16>(void* out, long i, const float* v) {
  *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(out) + i) =
      make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}
template <>
__device__ __forceinline__ void clip_store_vec<CLIP_F16>(void* out, long i, const float* v) {
  const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(out) + i) =
      make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}

// The values of one load that makes one 16-byte store: 16 bits to fp32 loads 8 bytes, so that a warp's
// stores are whole lines (with 16-byte loads each thread's two stores lie 16 bytes apart in 32: 266M
// bf16 gradients into fp32 took 286 us).
template <int T, int TO>
struct ClipLoad {
  static constexpr bool kHalf = T != CLIP_F32 && TO == CLIP_F32;
  static constexpr int N = kHalf ? 4 : ClipVec<T>::N;
  using V = std::conditional_t<kHalf, uint2, uint4>;
  static __device__ __forceinline__ void get(const uint4& u, float* v) { ClipVec<T>::get(u, v); }
  static __device__ __forceinline__ void get(const uint2& u, float* v) {
    float w[8];
    ClipVec<T>::get(make_uint4(u.x, u.y, 0u, 0u), w);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = w[j];
  }
};

template <int T, int TO>
__device__ __forceinline__ void clip_chunk_scale(const ClipDesc& d, int chunk, float f) {
  using L = ClipLoad<T, TO>;
  using V = typename L::V;
  constexpr int N = L::N, S = 16 / ClipVec<T>::N, SO = TO == CLIP_F32 ? 4 : 2;
  const ClipSpan s = clip_span<T>(d, chunk);
  const int vecs = (s.len - s.head) / N;
  const char* base = reinterpret_cast<const char*>(d.in) + s.lo * S;
  char* out = reinterpret_cast<char*>(d.out) + s.lo * SO;
  const V* p = reinterpret_cast<const V*>(base + s.head * S);
  char* o = out + s.head * SO;
  const bool wide = (reinterpret_cast<uintptr_t>(o) & (4 * SO - 1)) == 0;  // four outputs at a time
  const auto put = [&](int i, const V& u) {
    float v[N];
    L::get(u, v);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] *= f;
    if (wide) {
#pragma unroll
      for (int j = 0; j < N; j += 4) clip_store_vec<TO>(o, (long)i * N + j, v + j);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) clip_store(o, TO, (long)i * N + j, v[j]);
    }
  };
  constexpr int U = 4;
  int i = threadIdx.x;
  for (; i + (U - 1) * kClipThreads < vecs; i += U * kClipThreads) {
    V u[U];
#pragma unroll
    for (int j = 0; j < U; ++j) u[j] = __ldcs(p + i + j * kClipThreads);
#pragma unroll
    for (int j = 0; j < U; ++j) put(i + j * kClipThreads, u[j]);
  }
  for (; i < vecs; i += kClipThreads) put(i, __ldcs(p + i));
  for (int e = threadIdx.x; e < s.len - vecs * N; e += kClipThreads) {
    const int at = e < s.head ? e : e + vecs * N;
    clip_store(out, TO, at, clip_load(base, T, at) * f);
  }
}

template <int T>
__device__ __forceinline__ void clip_chunk_scale_to(const ClipDesc& d, int chunk, float f) {
  if (d.out_t == CLIP_F32) clip_chunk_scale<T, CLIP_F32>(d, chunk, f);
  else if (d.out_t == CLIP_BF16) clip_chunk_scale<T, CLIP_BF16>(d, chunk, f);
  else clip_chunk_scale<T, CLIP_F16>(d, chunk, f);
}

template <int CAP>
__global__ void __launch_bounds__(kClipThreads)
    clip_scale_kernel(const __grid_constant__ ClipList<CAP> l, const double* __restrict__ part, int np, float max_norm,
                      float* norm) {
  const float f = clip_total(part, np, max_norm, norm);
  // from the last chunk to the first: the norm has read the last ones last, so they are still in L2
  for (int c = l.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const ClipDesc& d = l.d[clip_find(l, c)];
    if (f == 1.f && d.in == d.out) continue;
    if (d.in_t == CLIP_F32) clip_chunk_scale_to<CLIP_F32>(d, c, f);
    else if (d.in_t == CLIP_BF16) clip_chunk_scale_to<CLIP_BF16>(d, c, f);
    else clip_chunk_scale_to<CLIP_F16>(d, c, f);
  }
}

__global__ void __launch_bounds__(kClipThreads)
    clip_scale_strided_kernel(const __grid_constant__ ClipStridedList l, const double* __restrict__ part, int np,
                              float max_norm) {
  const float f = clip_total(part, np, max_norm, nullptr);
  for (int t = 0; t < l.count; ++t) {
    const ClipStrided& d = l.d[t];
    if (f == 1.f && d.in == d.out) continue;
    for (long i = (long)blockIdx.x * kClipThreads + threadIdx.x; i < d.n; i += (long)gridDim.x * kClipThreads)
      clip_store(d.out, d.out_t, clip_offset(d.size, d.os, i),
                 clip_load(d.in, d.in_t, clip_offset(d.size, d.is, i)) * f);
  }
}

__global__ void __launch_bounds__(kClipThreads)
    clip_finish_kernel(const double* __restrict__ part, int np, float* norm) {
  clip_total(part, np, 0.f, norm);
}

// ------------------------------------------------------------------ host
static short clip_type(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CLIP_F32;
    case at::kBFloat16: return CLIP_BF16;
    case at::kHalf: return CLIP_F16;
    default: TORCH_CHECK(false, "clip_grads: fp32, bf16 or fp16 tensors expected, got ", t.scalar_type());
  }
}

static bool same_order(const at::Tensor& a, const at::Tensor& b) {
  for (int64_t k = 0; k < a.dim(); ++k)
    if (a.size(k) != 1 && a.stride(k) != b.stride(k)) return false;
  return true;
}

// Common dimensions of `a` and `b`, merged where both allow it; at most four are left.
static ClipStrided strided_desc(const at::Tensor& a, const at::Tensor* b) {
  ClipStrided d{};
  int nd = 0;
  for (int64_t k = 0; k < a.dim(); ++k) {
    const long sz = a.size(k), sa = a.stride(k), sb = b ? b->stride(k) : 0;
    if (sz == 1) continue;
    if (nd && d.is[nd - 1] == sa * sz && (!b || d.os[nd - 1] == sb * sz) && (long)d.size[nd - 1] * sz < (1L << 31)) {
      d.size[nd - 1] *= (int)sz;
      d.is[nd - 1] = sa;
      d.os[nd - 1] = sb;
      continue;
    }
    TORCH_CHECK(nd < 4, "clip_grads: a strided tensor of more than four dimensions that cannot be merged");
    TORCH_CHECK(sz < (1L << 31), "clip_grads: a strided tensor with a dimension over 2^31");
    d.size[nd] = (int)sz;
    d.is[nd] = sa;
    d.os[nd] = sb;
    ++nd;
  }
  for (int k = 3; k >= 0; --k) {  // the dimensions sit at the end
    const int from = k - (4 - nd);
    d.size[k] = from >= 0 ? d.size[from] : 1;
    d.is[k] = from >= 0 ? d.is[from] : 0;
    d.os[k] = from >= 0 ? d.os[from] : 0;
  }
  d.in = a.data_ptr();
  d.n = a.numel();
  d.in_t = clip_type(a);
  if (b) {
    d.out = b->data_ptr();
    d.out_t = clip_type(*b);
  }
  return d;
}

// Bytes that a tensor spans; `t`: the tensor where it leaves gaps between its elements, else null.
struct ClipRange {
  uintptr_t lo, hi;
  int i;
  bool out;
  const at::Tensor* t;
};

static MemView mem_view(const at::Tensor& t) {
  MemView v{reinterpret_cast<uintptr_t>(t.const_data_ptr()), (int)t.element_size(), {}, {}};
  for (int64_t k = 0; k < t.dim(); ++k) {
    v.size.push_back(t.size(k));
    v.stride.push_back(t.stride(k) * v.elem);
  }
  return v;
}
static MemView mem_view(const ClipRange& r) {
  return r.t ? mem_view(*r.t) : MemView{r.lo, 1, {(long)(r.hi - r.lo)}, {1}};
}

static ClipRange clip_range(const at::Tensor& t, bool dense, int i, bool out) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  if (dense) return {lo, lo + t.numel() * t.element_size(), i, out, nullptr};
  long last = 0;
  for (int64_t k = 0; k < t.dim(); ++k) last += (t.size(k) - 1) * t.stride(k);
  return {lo, lo + (last + 1) * t.element_size(), i, out, &t};
}

// Outputs must not overlap one another, nor any input; a tensor scaled in place has one range.  Ranges
// that meet are looked at closer where one of them has gaps: interleaved views share no element.
static void check_ranges(std::vector<ClipRange>& r) {
  const auto less = [](const ClipRange& a, const ClipRange& b) { return a.lo < b.lo; };
  if (!std::is_sorted(r.begin(), r.end(), less)) std::sort(r.begin(), r.end(), less);
  uintptr_t hi = 0;
  bool meet = false;
  for (const auto& x : r) {
    meet |= x.lo < hi;
    hi = std::max(hi, x.hi);
  }
  if (!meet) return;
  std::vector<std::pair<const ClipRange*, MemView>> open;  // those that reach past the start of the present one
  for (const auto& x : r) {
    open.erase(std::remove_if(open.begin(), open.end(), [&](const auto& o) { return o.first->hi <= x.lo; }), open.end());
    MemView v = mem_view(x);
    for (const auto& [y, w] : open) {
      if (!x.out && !y->out) continue;
      const bool apart = (x.t || y->t) && !views_overlap(v, w);
      TORCH_CHECK(apart || x.i == y->i, "clip_grads: tensors ", y->i, " and ", x.i, " overlap in memory");
      TORCH_CHECK(apart, "clip_grads: output ", x.i, " overlaps its gradient in memory without being it");
    }
    open.emplace_back(&x, std::move(v));
  }
}

template <int CAP>
static void launch_lists(const std::vector<ClipDesc>& all, size_t at, size_t count, int grid, bool scale, double* part,
                         int np, float max_norm, float* norm, cudaStream_t st) {
  ClipList<CAP> l;
  l.count = (int)count;
  l.chunks = 0;
  for (size_t k = 0; k < count; ++k) {
    l.d[k] = all[at + k];
    l.d[k].first = l.chunks;
    l.chunks += (int)((l.d[k].n + kClipChunk - 1) / kClipChunk);
  }
  if (scale) clip_scale_kernel<CAP><<<grid, kClipThreads, 0, st>>>(l, part, np, max_norm, norm);
  else clip_norm_kernel<CAP><<<grid, kClipThreads, 0, st>>>(l, part);
  count_launch();
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// The norm (fp32 scalar) of the tensors `in` together (those that are there); with `scale`
// also in[i] *= factor or, with `out` (aligned with `in`, of the same shapes),
// out[i] = in[i] * factor (0 where there is no in[i]).  out[i] may be in[i].
at::Tensor clip_grads(std::vector<std::optional<at::Tensor>> in,
                      std::optional<std::vector<std::optional<at::Tensor>>> out, double max_norm, bool scale) {
  TORCH_CHECK_VALUE(max_norm >= 0.0, "clip_grads: max_norm must not be negative, got ", max_norm);
  TORCH_CHECK_VALUE(!out || out->size() == in.size(), "clip_grads: ", in.size(), " gradients but ",
                    out ? out->size() : 0, " outputs");
  const at::Tensor* head = nullptr;
  for (const auto& t : in)
    if (t) {
      head = &*t;
      break;
    }
  TORCH_CHECK_VALUE(head, "clip_grads: an empty list has no device");
  const auto dev = head->device();
  TORCH_CHECK(dev.is_cuda(), "clip_grads: CUDA tensors expected");
  c10::cuda::CUDAGuard guard(dev);
  std::vector<ClipDesc> dense;
  std::vector<ClipStrided> strided;
  std::vector<ClipRange> ranges;
  dense.reserve(in.size());
  if (scale) ranges.reserve(out ? 2 * in.size() : in.size());
  std::vector<const at::Tensor*> absent;  // outputs without a gradient
  for (size_t i = 0; i < in.size(); ++i) {
    if (!in[i]) {
      if (scale && out && (*out)[i] && (*out)[i]->numel()) {
        const at::Tensor& b = *(*out)[i];
        TORCH_CHECK(b.device() == dev, "clip_grads: tensor ", i, " is on another device");
        ranges.push_back(clip_range(b, b.is_non_overlapping_and_dense(), (int)i, true));
        absent.push_back(&b);
      }
      continue;
    }
    const at::Tensor& a = *in[i];
    TORCH_CHECK_VALUE(!scale || !out || (*out)[i], "clip_grads: every gradient needs an output of its own shape");
    const at::Tensor* b = !scale ? nullptr : out ? &*(*out)[i] : &a;
    TORCH_CHECK(a.device() == dev && (!b || b->device() == dev), "clip_grads: tensor ", i, " is on another device");
    const short ta = clip_type(a), tb = !b ? 0 : b == &a ? ta : clip_type(*b);
    TORCH_CHECK_VALUE(!b || b == &a || b->sizes() == a.sizes(), "clip_grads: output ", i,
                      " has another shape than its gradient");
    const long numel = a.numel();
    if (numel == 0) continue;
    const void* pa = a.const_data_ptr();
    void* pb = b ? b->mutable_data_ptr() : nullptr;
    const bool same = pa == pb;
    TORCH_CHECK(!same || (ta == tb && same_order(a, *b)), "clip_grads: output ", i, " overlays its gradient differently");
    const bool dense_a = a.is_non_overlapping_and_dense();
    const bool dense_b = b && (b == &a ? dense_a : b->is_non_overlapping_and_dense());
    const bool flat = dense_a && (!b || same || (dense_b && same_order(a, *b)));
    if (b) {
      TORCH_CHECK(dense_b || !view_overlaps_itself(mem_view(*b)), "clip_grads: output ", i, " overlaps itself");
      if (!same) ranges.push_back(clip_range(a, dense_a, (int)i, false));
      ranges.push_back(clip_range(*b, dense_b, (int)i, true));
    }
    if (flat) dense.push_back({pa, pb, numel, 0, ta, tb});
    else strided.push_back(strided_desc(a, b));
  }
  check_ranges(ranges);
  for (const at::Tensor* b : absent) b->zero_();

  // launches: lists of at most 960 tensors, each with a grid fixed by its number of chunks
  struct Part { size_t at, count; int grid; };
  std::vector<Part> parts;
  int np = 0;
  for (size_t at = 0; at < dense.size();) {
    Part p{at, 0, 0};
    long chunks = 0;
    while (at < dense.size() && p.count < 960) {
      const long c = (dense[at].n + kClipChunk - 1) / kClipChunk;
      if (p.count && chunks + c >= (1L << 31)) break;
      chunks += c;
      ++p.count;
      ++at;
    }
    TORCH_CHECK(chunks < (1L << 31), "clip_grads: a tensor of over 2^43 elements");
    p.grid = (int)std::min<long>(chunks, kClipGrid);
    np += p.grid;
    parts.push_back(p);
  }
  const size_t nlists = (strided.size() + kClipStridedMax - 1) / kClipStridedMax;
  np += (int)nlists * kClipGrid;
  auto norm = at::empty({}, head->options().dtype(at::kFloat));
  auto part = at::empty({std::max(np, 1)}, head->options().dtype(at::kDouble));
  double* pp = part.data_ptr<double>();
  float* nn = norm.data_ptr<float>();
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  for (int pass = 0; pass < (scale ? 2 : 1); ++pass) {
    double* to = pp;
    bool first = true;
    for (const auto& p : parts) {
      double* q = pass ? pp : to;
      float* wr = pass && first ? nn : nullptr;
      if (p.count <= 32) launch_lists<32>(dense, p.at, p.count, p.grid, pass, q, np, (float)max_norm, wr, st);
      else if (p.count <= 256) launch_lists<256>(dense, p.at, p.count, p.grid, pass, q, np, (float)max_norm, wr, st);
      else launch_lists<960>(dense, p.at, p.count, p.grid, pass, q, np, (float)max_norm, wr, st);
      to += p.grid;
      first = false;
    }
    for (size_t s = 0; s < nlists; ++s) {
      ClipStridedList l;
      l.count = (int)std::min<size_t>(kClipStridedMax, strided.size() - s * kClipStridedMax);
      std::copy_n(strided.begin() + s * kClipStridedMax, l.count, l.d);
      if (pass) clip_scale_strided_kernel<<<kClipGrid, kClipThreads, 0, st>>>(l, pp, np, (float)max_norm);
      else clip_norm_strided_kernel<<<kClipGrid, kClipThreads, 0, st>>>(l, to);
      to += kClipGrid;
      count_launch();
      C10_CUDA_KERNEL_LAUNCH_CHECK();
    }
  }
  if (!scale || parts.empty()) {
    clip_finish_kernel<<<1, kClipThreads, 0, st>>>(pp, np, nn);
    count_launch();
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return norm;
}

}  // namespace dtb
