// gfd_rowops.h -- element types and wave helpers of the row-wise training
// operators (gfd_adam.hip, gfd_class_logp.hip, gfd_group_norm.hip): fp32, bf16
// and fp16 elements read and written in vectors, arithmetic in fp32 or fp64.
#pragma once

#include <type_traits>

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

// V elements read as one access and kept in as many registers as they fill (an array of 16-bit
// elements takes one each)
template <typename T, int V>
struct Raw {
  static constexpr int kWords = (V * int(sizeof(T)) + 3) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void read(const T* p) {
    if constexpr (V * sizeof(T) < 4) {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    } else {
      const auto v = *reinterpret_cast<const Pack<uint32_t, kWords>*>(p);
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = v.v[i];
    }
  }
  __device__ __forceinline__ float at(int j) const {  // j: a constant after unrolling
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[j]);
    } else if constexpr (std::is_same<T, bf16_t>::value) {
      return __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
    } else {
      union {
        uint16_t u;
        T f;
      } h;
      h.u = uint16_t(j & 1 ? w[j / 2] >> 16 : w[j / 2]);
      return to_f32(h.f);
    }
  }
};

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
