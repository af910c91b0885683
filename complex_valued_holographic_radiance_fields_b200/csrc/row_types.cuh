// Element types and row layouts shared by the row kernels (row_tables.cu, row_moves.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace cvhrf {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// VEC consecutive elements, moved by one load or store of sizeof(T) * VEC bytes.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

inline size_t row_type_bytes(int dtype) { return dtype == CVHRF_F32 ? 4 : 2; }
inline bool row_type_ok(int dtype) { return dtype == CVHRF_F32 || dtype == CVHRF_BF16 || dtype == CVHRF_F16; }
inline int next_pow2(int x) {
  int p = 1;
  while (p < x) p <<= 1;
  return p;
}

// Whether rows of `width` elements every `stride` elements from p can be moved 16 bytes at a
// time (torch's own allocations are aligned; slices and odd widths need not be).
inline bool rows_16(const void* p, long long stride, int width, size_t elem) {
  return ((uintptr_t)p & 15) == 0 && (stride * (long long)elem) % 16 == 0 && ((size_t)width * elem) % 16 == 0;
}

}  // namespace cvhrf
