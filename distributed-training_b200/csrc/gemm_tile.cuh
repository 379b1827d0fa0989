// Tile helpers shared by the tcgen05 GEMMs (gemm.cu: dense, moe.cu: grouped by expert):
// tile sizes, the order of output tiles, the epilogue's staging slabs, and the
// tensor maps of operands and outputs.
#pragma once

#include <c10/util/Exception.h>

#include <mutex>

#include "common.cuh"

namespace dtb {

constexpr int kBM = 128;
constexpr int kBK = 64;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + kEpiWarps * 32;
constexpr int kEpiSlab = 4096;  // bytes of store staging per epilogue warp (32 rows x 32 fp32)

__device__ __forceinline__ void tile_coords(int t, int mt, int nt, int& mi, int& ni) {
  // Group 16 M-tiles together so CTAs running concurrently share B (and A) tiles in L2.
  const int G = 16;
  const int per_group = G * nt;
  const int g = t / per_group;
  const int first = g * G;
  const int gm = min(G, mt - first);
  const int r = t - g * per_group;
  mi = first + r % gm;
  ni = r / gm;
}

__device__ __forceinline__ void load_bf16x8(const bf16* src, float* v) {
  uint4 u = *reinterpret_cast<const uint4*>(src);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f = __bfloat1622float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// Load 32 bf16 values [col, col+32) of a row into fp32 (zeros past n_valid).
__device__ __forceinline__ void load_row32(const bf16* rowp, int col, int N, float* v) {
  if (col + 32 <= N) {
#pragma unroll
    for (int j = 0; j < 32; j += 8) load_bf16x8(rowp + col + j, v + j);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = (col + j < N) ? bf2f(rowp[col + j]) : 0.f;
  }
}

// Staging slabs hold one 32x32 output chunk, one row per lane, in the layout of the
// TMA store's swizzle mode, so that a warp's 16-byte stores hit distinct banks:
//   bf16 rows (64 B, SWIZZLE_64B):   16-byte unit j of row r sits at unit j ^ ((r >> 1) & 3)
//   fp32 rows (128 B, SWIZZLE_128B): 16-byte unit j of row r sits at unit j ^ (r & 7)
// (unswizzled rows 64 / 128 B apart put 8 lanes of a store phase on 2 / 1 bank groups:
// 4- and 8-way conflicts).  Slabs start on 2 KB boundaries, a multiple of both
// patterns' periods (512 B and 1 KB), as the swizzled TMA store requires.
__device__ __forceinline__ int slab_unit_bf16(int lane, int j) { return j ^ ((lane >> 1) & 3); }
__device__ __forceinline__ int slab_unit_f32(int lane, int j) { return j ^ (lane & 7); }

// Write 32 fp32 values as bf16 into this lane's 64-byte row of a slab.
__device__ __forceinline__ void slab_put_bf16(uint8_t* slab, int lane, const float* v) {
  uint4* dst = reinterpret_cast<uint4*>(slab + lane * 64);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint4 u;
    u.x = pack_bf16x2(v[8 * j + 0], v[8 * j + 1]);
    u.y = pack_bf16x2(v[8 * j + 2], v[8 * j + 3]);
    u.z = pack_bf16x2(v[8 * j + 4], v[8 * j + 5]);
    u.w = pack_bf16x2(v[8 * j + 6], v[8 * j + 7]);
    dst[slab_unit_bf16(lane, j)] = u;
  }
}

__device__ __forceinline__ void slab_put_f32(uint8_t* slab, int lane, const float* v) {
  float4* dst = reinterpret_cast<float4*>(slab + lane * 128);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    dst[slab_unit_f32(lane, j)] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
}

// Before packing a chunk: lane 0 waits until the store that last used this (sub-)slab
// has read it - with two halves that is every store but the most recent one.
__device__ __forceinline__ void epi_slab_acquire(int lane, bool dbl) {
  if (lane == 0) {
    if (dbl) bulk_wait_read1();
    else bulk_wait_read0();
  }
  __syncwarp();
}

// ------------------------------------------------------------------ host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn get_encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
    TORCH_CHECK(e == cudaSuccess && q == cudaDriverEntryPointSuccess && p, "cuTensorMapEncodeTiled unavailable");
    fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// 2-D bf16 operand map over a row-major matrix [rows, cols] with row stride ld (elements), 128B swizzle.
inline CUtensorMap make_map(const void* base, long rows, long cols, long ld, int box_cols, int box_rows) {
  CUtensorMap m;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = get_encode_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box,
                               estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code ", (int)r);
  return m;
}

// Store map: [rows, cols] (optionally [depth, rows, cols]) row-major, 32x32 boxes, with
// the staging slabs' swizzle (64B for bf16 rows, 128B for fp32 rows).
inline CUtensorMap make_store_map(void* base, bool f32, long rows, long cols, long ld, long depth = 0) {
  CUtensorMap m;
  const int esz = f32 ? 4 : 2;
  const CUtensorMapDataType dt = f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapSwizzle sw = f32 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r;
  if (depth > 0) {
    cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)depth};
    cuuint64_t strides[2] = {(cuuint64_t)ld * esz, (cuuint64_t)ld * rows * esz};
    cuuint32_t box[3] = {32, 32, 1};
    r = get_encode_fn()(&m, dt, 3, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        sw, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  } else {
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * esz};
    cuuint32_t box[2] = {32, 32};
    r = get_encode_fn()(&m, dt, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        sw, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  }
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled (store) failed with code ", (int)r);
  return m;
}

inline int num_sms() {
  static int n = 0;
  if (!n) {
    int dev;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  }
  return n;
}

}  // namespace dtb
