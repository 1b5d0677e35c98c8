// gfd_adam.hip -- one Adam / AdamW step over many tensors at once (the
// optimizer of the reference's training loop, train.py:353), states in fp32 or
// in 8 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p -= lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory: 28 B an element (fp32 parameters and states), 10 B and the
// scales (16-bit parameters, 8-bit states); the step is one launch for up to
// kMaxTensors tensors, whose pointers travel in the kernel arguments (no copy to
// the device, so a captured call holds them too).
//   * Work is cut into chunks of kChunk elements of one tensor; a block takes
//     chunks blockIdx, blockIdx + gridDim, ...  A chunk's tensor is the number of
//     first-chunk entries not above it: two ballots over the table, which the
//     lanes of a wave hold.
//   * The step count lives on the device.  Every block reads it, the last block
//     to arrive at the ticket advances it: no second launch, and no argument
//     that changes from step to step.
//   * 8 elements a lane: 32 lanes hold a block of 256, so its two largest
//     magnitudes are five lane exchanges each.
#include "gfd_rowops.h"

using namespace gfd;

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 8;                     // elements a thread
constexpr int kChunk = kThreads * kPer;     // 2048: a multiple of the 256-element state blocks
constexpr int kStateBlock = 256;
constexpr int kMaxTensors = 96;             // the argument block stays under 4 KB
constexpr int kMaxBlocks = 2048;            // 8 blocks a CU

struct AdamTensor {
  void* p;
  const void* g;
  int64_t numel;
  int64_t first;
  int32_t slot;
  uint32_t chunk0;  // chunks of the tensors before it
};

struct AdamArgs {
  AdamTensor t[kMaxTensors];
  void* m;
  void* v;
  float* ms;
  float* vs;
  int32_t* step;
  const float* lr_dev;
  uint32_t* ticket;
  double b1, b2, lr, wd;
  float eps;
  uint32_t seed;
  uint32_t chunks;
  int n;
  int decoupled;
};
static_assert(sizeof(AdamArgs) <= 4096, "kernel arguments");

// b^t by squaring (fp64: the relative error grows as t 2^-53)
__device__ double power(double b, uint32_t t) {
  double r = 1.0;
  for (; t; t >>= 1) {
    if (t & 1) r *= b;
    b *= b;
  }
  return r;
}

// 32-bit hash: two multiplications between shifts
__device__ __forceinline__ uint32_t mix32(uint32_t h) {
  h ^= h >> 16;
  h *= 0x7FEB352Du;
  h ^= h >> 15;
  h *= 0x846CA68Bu;
  return h ^ (h >> 16);
}

// The e4m3 code of x * inv (inv a power of two, |x * inv| < 256 for finite x) by
// stochastic rounding: 16 random bits are added to the 20 mantissa bits that the
// code drops (aligned with the highest of them) and the rest is cut off.  Below
// 2^-6, the smallest normal, codes step by 2^-9 as they do in [2^-6, 2^-5): the
// same cut after 2^-6 is added, 8 codes lower.
template <bool FLOOR>
__device__ __forceinline__ uint32_t encode(float x, float inv, uint32_t u16) {
  const float t = x * inv;
  const float a = fabsf(t);
  const bool low = a < 0.015625f;
  const float z = low ? a + 0.015625f : a;
  uint32_t c = ((__float_as_uint(z) + (u16 << 4)) >> 20) - (low ? (120u << 3) + 8u : 120u << 3);
  if (FLOOR) c = (c == 0 && a > 0.f) ? 1u : c;
  c = a < 512.f ? c : 0x7Fu;  // NaN and infinity (false for both): the NaN code
  return c | (__float_as_uint(t) >> 31 << 7);
}

// the scale 2^e of a block whose largest finite magnitude is a: a / 2^e in [128, 256)
__device__ __forceinline__ float scale_of(float a) {
  const int e = int(__float_as_uint(a) >> 23) - 7;
  return __uint_as_float(uint32_t(e < 27 ? 27 : e) << 23);  // 2^-100 at least
}
__device__ __forceinline__ float inverse_pow2(float s) {
  return __uint_as_float((254u << 23) - __float_as_uint(s));
}

// a b + c d, each product rounded: where they cancel the sum is 0, not a product's rounding
__device__ __forceinline__ double two_products(double a, double b, double c, double d) {
#pragma clang fp contract(off)
  return a * b + c * d;
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < __builtin_inff() ? a : 0.f;
}

// max over the 32 lanes that share a state block
__device__ __forceinline__ float max32(float v) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

template <typename T, int BITS>
__global__ void __launch_bounds__(kThreads) k_adam(const AdamArgs a) {
  const int lane = threadIdx.x & 63;
  const uint32_t c0 = lane < a.n ? a.t[lane].chunk0 : ~0u;
  const uint32_t c1 = lane + 64 < a.n ? a.t[lane + 64].chunk0 : ~0u;
  const double lr = a.lr_dev ? double(*a.lr_dev) : a.lr;
  const float keep = a.decoupled ? float(1.0 - lr * a.wd) : 1.f;
  const double l2 = a.decoupled ? 0.0 : a.wd;
  int was = -1;
  float rate = 0.f, unbias = 0.f;
  uint32_t key = 0;
  for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
    const int i = wave_uniform(__popcll(__ballot(c0 <= chunk)) + __popcll(__ballot(c1 <= chunk)) - 1);
    const AdamTensor& t = a.t[i];
    if (i != was) {
      was = i;
      const uint32_t now = uint32_t(a.step[t.slot]) + 1u;
      rate = float(lr / (1.0 - power(a.b1, now)));
      unbias = float(1.0 / sqrt(1.0 - power(a.b2, now)));
      key = mix32(mix32(now) + a.seed);
    }
    const int64_t at = int64_t(chunk - t.chunk0) * kChunk + threadIdx.x * kPer;
    const int64_t left = t.numel - at;  // elements of this thread, if positive
    const int64_t e = t.first + at;
    T* pp = static_cast<T*>(t.p) + at;
    const T* gp = static_cast<const T*>(t.g) + at;
    constexpr int kV = 16 / sizeof(T) < kPer ? 16 / sizeof(T) : kPer;
    const bool whole = left >= kPer &&
                       ((reinterpret_cast<uintptr_t>(pp) | reinterpret_cast<uintptr_t>(gp)) & 15) == 0;
    float p[kPer], g[kPer];
    if (whole) {
#pragma unroll
      for (int j = 0; j < kPer; j += kV) {
        const auto pv = *reinterpret_cast<const Pack<T, kV>*>(pp + j);
        const auto gv = *reinterpret_cast<const Pack<T, kV>*>(gp + j);
#pragma unroll
        for (int k = 0; k < kV; ++k) {
          p[j + k] = to_f32(pv.v[k]);
          g[j + k] = to_f32(gv.v[k]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        p[j] = j < left ? to_f32(pp[j]) : 0.f;
        g[j] = j < left ? to_f32(gp[j]) : 0.f;
      }
    }
    if (BITS == 32) {
      float* mp = static_cast<float*>(a.m) + e;
      float* vp = static_cast<float*>(a.v) + e;
      const float b1 = float(a.b1), b2 = float(a.b2), d1 = float(1.0 - a.b1), d2 = float(1.0 - a.b2);
      float m[kPer], v[kPer];
      if (left >= kPer) {
#pragma unroll
        for (int j = 0; j < kPer; j += 4) {
          *reinterpret_cast<Pack<float, 4>*>(m + j) = *reinterpret_cast<const Pack<float, 4>*>(mp + j);
          *reinterpret_cast<Pack<float, 4>*>(v + j) = *reinterpret_cast<const Pack<float, 4>*>(vp + j);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          m[j] = j < left ? mp[j] : 0.f;
          v[j] = j < left ? vp[j] : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const float gj = g[j] + float(l2) * p[j];
        m[j] = b1 * m[j] + d1 * gj;
        v[j] = b2 * v[j] + d2 * gj * gj;
        p[j] = p[j] * keep - rate * (m[j] / (sqrtf(v[j]) * unbias + a.eps));
      }
      if (left >= kPer) {
#pragma unroll
        for (int j = 0; j < kPer; j += 4) {
          *reinterpret_cast<Pack<float, 4>*>(mp + j) = *reinterpret_cast<const Pack<float, 4>*>(m + j);
          *reinterpret_cast<Pack<float, 4>*>(vp + j) = *reinterpret_cast<const Pack<float, 4>*>(v + j);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          if (j < left) {
            mp[j] = m[j];
            vp[j] = v[j];
          }
        }
      }
    } else {
      uint8_t* mp = static_cast<uint8_t*>(a.m) + e;
      uint8_t* vp = static_cast<uint8_t*>(a.v) + e;
      uint32_t mc[2] = {0, 0}, vc[2] = {0, 0};
      float ms = 0.f, vs = 0.f;
      if (left > 0) {
        ms = a.ms[e / kStateBlock];
        vs = a.vs[e / kStateBlock];
      }
      if (left >= kPer) {
        *reinterpret_cast<Pack<uint32_t, 2>*>(mc) = *reinterpret_cast<const Pack<uint32_t, 2>*>(mp);
        *reinterpret_cast<Pack<uint32_t, 2>*>(vc) = *reinterpret_cast<const Pack<uint32_t, 2>*>(vp);
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          if (j < left) {
            mc[j / 4] |= uint32_t(mp[j]) << 8 * (j & 3);
            vc[j / 4] |= uint32_t(vp[j]) << 8 * (j & 3);
          }
        }
      }
      float m[kPer], r[kPer];
      float mmax = 0.f, rmax = 0.f;
      const double d1 = 1.0 - a.b1, d2 = 1.0 - a.b2;
      auto decode = [](uint32_t w, int j) {  // (the byte index has to be a literal)
        switch (j & 3) {
          case 0: return __builtin_amdgcn_cvt_f32_fp8(int(w), 0);
          case 1: return __builtin_amdgcn_cvt_f32_fp8(int(w), 1);
          case 2: return __builtin_amdgcn_cvt_f32_fp8(int(w), 2);
          default: return __builtin_amdgcn_cvt_f32_fp8(int(w), 3);
        }
      };
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const double old_m = double(decode(mc[j / 4], j) * ms);
        const double old_r = double(decode(vc[j / 4], j) * vs);
        // fp64, so that a moment next to a border between two scales or codes falls on its side
        const double gj = two_products(double(g[j]), 1.0, l2, double(p[j]));
        m[j] = float(two_products(a.b1, old_m, d1, gj));
        r[j] = sqrtf(float(two_products(a.b2, old_r * old_r, d2, gj * gj)));
        p[j] = p[j] * keep - rate * (m[j] / (r[j] * unbias + a.eps));
        mmax = fmaxf(mmax, finite_abs(m[j]));
        rmax = fmaxf(rmax, finite_abs(r[j]));
      }
      ms = scale_of(max32(mmax));
      vs = scale_of(max32(rmax));
      const float mi = inverse_pow2(ms), vi = inverse_pow2(vs);
      const uint32_t k2 = (e >> 32) ? key ^ mix32(uint32_t(e >> 32)) : key;
      mc[0] = mc[1] = vc[0] = vc[1] = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const uint32_t u = mix32(uint32_t(e + j) * 0x9E3779B1u + k2);
        mc[j / 4] |= encode<false>(m[j], mi, u & 0xFFFFu) << 8 * (j & 3);
        vc[j / 4] |= encode<true>(r[j], vi, u >> 16) << 8 * (j & 3);
      }
      if (left >= kPer) {
        *reinterpret_cast<Pack<uint32_t, 2>*>(mp) = *reinterpret_cast<const Pack<uint32_t, 2>*>(mc);
        *reinterpret_cast<Pack<uint32_t, 2>*>(vp) = *reinterpret_cast<const Pack<uint32_t, 2>*>(vc);
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          if (j < left) {
            mp[j] = uint8_t(mc[j / 4] >> 8 * (j & 3));
            vp[j] = uint8_t(vc[j / 4] >> 8 * (j & 3));
          }
        }
      }
      if (left > 0 && (threadIdx.x & 31) == 0) {
        a.ms[e / kStateBlock] = ms;
        a.vs[e / kStateBlock] = vs;
      }
    }
    if (whole) {
#pragma unroll
      for (int j = 0; j < kPer; j += kV) {
        Pack<T, kV> pv;
#pragma unroll
        for (int k = 0; k < kV; ++k) pv.v[k] = from_f32<T>(p[j + k]);
        *reinterpret_cast<Pack<T, kV>*>(pp + j) = pv;
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (j < left) pp[j] = from_f32<T>(p[j]);
    }
  }
  // every block has read the step counts it needs: the last one here advances them
  __shared__ uint32_t last;
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(a.ticket, 1u) == gridDim.x - 1 ? 1u : 0u;
  __syncthreads();
  if (last) {
    for (int i = threadIdx.x; i < a.n; i += kThreads) a.step[a.t[i].slot] += 1;
    if (threadIdx.x == 0) *a.ticket = 0u;
  }
}

}  // namespace

extern "C" {

gfd_status gfd_adam_step(const gfd_adam_tensor* tensors, int64_t num_tensors, int dtype,
                         int state_bits, void* exp_avg, void* exp_avg_sq, float* exp_avg_scale,
                         float* exp_avg_sq_scale, int32_t* step, double lr,
                         const float* lr_device, double beta1, double beta2, double eps,
                         double weight_decay, int decoupled, uint32_t seed, uint32_t* ticket,
                         gfd_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (num_tensors < 0 || !float_dtype(dtype)) return GFD_ERR_ARGUMENT;
  if (state_bits != 32 && state_bits != 8) return GFD_ERR_UNSUPPORTED;
  if (num_tensors == 0) return GFD_OK;
  if (!tensors || !exp_avg || !exp_avg_sq || !step || !ticket) return GFD_ERR_ARGUMENT;
  if (state_bits == 8 && (!exp_avg_scale || !exp_avg_sq_scale)) return GFD_ERR_ARGUMENT;
  if (!aligned_to(exp_avg, 16) || !aligned_to(exp_avg_sq, 16)) return GFD_ERR_ARGUMENT;
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0))
    return GFD_ERR_ARGUMENT;
  for (int64_t i = 0; i < num_tensors; ++i) {
    const gfd_adam_tensor& t = tensors[i];
    if (t.numel < 0 || t.numel > (int64_t(1) << 40) || t.first < 0 || t.first % kStateBlock ||
        t.slot < 0 || t.slot > INT32_MAX)
      return GFD_ERR_ARGUMENT;
    if (t.numel > 0 && (!t.param || !t.grad)) return GFD_ERR_ARGUMENT;
    if (!aligned_to(t.param, dtype_size(dtype)) || !aligned_to(t.grad, dtype_size(dtype)))
      return GFD_ERR_ARGUMENT;
  }
  for (int64_t i0 = 0; i0 < num_tensors; i0 += kMaxTensors) {
    AdamArgs a;
    a.n = int(num_tensors - i0 < kMaxTensors ? num_tensors - i0 : kMaxTensors);
    int64_t chunks = 0;
    for (int i = 0; i < a.n; ++i) {
      const gfd_adam_tensor& t = tensors[i0 + i];
      a.t[i] = {t.param, t.grad, t.numel, t.first, int32_t(t.slot), uint32_t(chunks)};
      chunks += (t.numel + kChunk - 1) / kChunk;
    }
    if (chunks >= (int64_t(1) << 31)) return GFD_ERR_UNSUPPORTED;
    a.m = exp_avg;
    a.v = exp_avg_sq;
    a.ms = exp_avg_scale;
    a.vs = exp_avg_sq_scale;
    a.step = step;
    a.lr_dev = lr_device;
    a.ticket = ticket;
    a.b1 = beta1;
    a.b2 = beta2;
    a.lr = lr;
    a.wd = weight_decay;
    a.eps = float(eps);
    a.seed = seed;
    a.chunks = uint32_t(chunks);
    a.decoupled = decoupled != 0;
    const int grid = int(chunks < 1 ? 1 : chunks < kMaxBlocks ? chunks : kMaxBlocks);
    const gfd_status st = with_dtype(dtype, [&](auto tag) {
      using T = decltype(tag);
      if (state_bits == 32)
        k_adam<T, 32><<<grid, kThreads, 0, stream>>>(a);
      else
        k_adam<T, 8><<<grid, kThreads, 0, stream>>>(a);
      GFD_LAUNCH_CHECK();
      return GFD_OK;
    });
    if (st != GFD_OK) return st;
  }
  return GFD_OK;
}

}  // extern "C"
