// Shared by the sequence-network operators (recurrence.cu, norm.cu, adamw.cu):
// element types, vector loads and stores, and the entry points' error returns.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/cpab_b200.h"
#include "launch.h"

namespace cpab {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// The two 16-bit elements of a word as float32, and two values rounded to one.
template <typename T>
__device__ __forceinline__ float2 unpack_pair(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack_pair<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 unpack_pair<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&p);
}
template <>
__device__ __forceinline__ uint32_t pack_pair<__half>(float a, float b) {
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&p);
}
// The rounded sums of two words' elements (one rounding, as of the float32 sum).
template <typename T>
__device__ __forceinline__ uint32_t add_pair(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t add_pair<__nv_bfloat16>(uint32_t a, uint32_t b) {
  const __nv_bfloat162 s = __hadd2(*reinterpret_cast<const __nv_bfloat162 *>(&a),
                                   *reinterpret_cast<const __nv_bfloat162 *>(&b));
  return *reinterpret_cast<const uint32_t *>(&s);
}
template <>
__device__ __forceinline__ uint32_t add_pair<__half>(uint32_t a, uint32_t b) {
  const __half2 s = __hadd2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
  return *reinterpret_cast<const uint32_t *>(&s);
}

// N consecutive elements moved by one access of N * sizeof(T) bytes (at most
// 16), which is also the alignment it needs.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

// Rows the vector kernels may take: base and row stride multiples of `bytes`.
inline bool aligned_to(const void *p, int64_t stride_elems, int elem_size, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (stride_elems * elem_size) % bytes == 0;
}

inline int dtype_size(int dtype) { return dtype == CPAB_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) {
  return dtype == CPAB_F32 || dtype == CPAB_F16 || dtype == CPAB_BF16;
}

// Status of a launch: 0 clears this thread's message.
inline int launch_status(cudaError_t e, const char *what) {
  if (e == cudaSuccess) return report_error(CPAB_OK, "%s", "");
  return report_error(CPAB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

}  // namespace cpab
