// gfd_rowops.h -- element types and wave helpers of the row-wise training
// operators (gfd_adam.hip, gfd_class_logp.hip, gfd_group_norm.hip): fp32, bf16
// and fp16 elements read and written in vectors, arithmetic in fp32 or fp64.
#pragma once

#include "gfd_common.h"

namespace gfd {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// V elements read or written as one access (V * sizeof(T) <= 16)
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

// conversions through fp32; the narrowing ones round to nearest even
template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  return static_cast<T>(v);
}

inline bool aligned_to(const void* p, size_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

inline bool float_dtype(int dtype) {
  return dtype == GFD_DTYPE_F32 || dtype == GFD_DTYPE_BF16 || dtype == GFD_DTYPE_F16;
}

inline size_t dtype_size(int dtype) { return dtype == GFD_DTYPE_F32 ? 4 : 2; }

// f(tag of the element type) for a dtype that float_dtype accepts
template <typename F>
gfd_status with_dtype(int dtype, F f) {
  if (dtype == GFD_DTYPE_BF16) return f(bf16_t{});
  if (dtype == GFD_DTYPE_F16) return f(f16_t{});
  return f(float{});
}

}  // namespace gfd
