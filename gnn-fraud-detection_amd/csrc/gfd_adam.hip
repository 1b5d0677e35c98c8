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
//     to arrive advances it: no second launch, and no argument that changes from
//     step to step.  Blocks arrive at kLeaves counters a cache line apart, the
//     last ones of those at a root: a thousand blocks at one counter take
//     15 us to pass it.
//   * 8 elements a lane: 32 lanes hold a block of 256, so its two largest
//     magnitudes are five lane exchanges each.  8-bit states are bound by the
//     memory and the arithmetic together (64 operations an element, 12 of them
//     fp64): 160M elements with bf16 parameters 398 us, 4.0 TB/s; the same reads
//     and writes alone take 337 us.
#include "gfd_rowops.h"

using namespace gfd;

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 8;                     // elements a thread
constexpr int kChunk = kThreads * kPer;     // 2048: a multiple of the 256-element state blocks
constexpr int kStateBlock = 256;
constexpr int kMaxTensors = 96;             // the argument block stays under 4 KB
// waves a SIMD that the registers have to allow: 32-bit states 7 (72 registers), 8-bit ones 6
// (80; at 160M elements 5 take 415 us, 6 398 us, 7, with spills, 423 us)
constexpr int kWaves32 = 7, kWaves8 = 6;
// 32-bit states: a block a chunk (120M elements: 645 us, 5.2 TB/s; 687 us with as many blocks as
// fit the card, each with many chunks).  8-bit states, whose set-up weighs more beside their
// fewer bytes: as many blocks as fit (398 us against 415 us)
constexpr int kMaxBlocks32 = 1 << 20, kMaxBlocks8 = 256 * kWaves8;
constexpr int kLeaves = 32;                 // arrival counters, kLine apart, and a root behind them
constexpr int kLine = 32;
static_assert((kLeaves + 1) * kLine == GFD_ADAM_TICKETS, "arrival counters");

constexpr uint32_t kInfBits = 0x7F800000u;

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

// 32-bit hash: two multiplications between shifts, with constants of C. Wellons' published search
// for the least bias between input and output bits
__device__ __forceinline__ uint32_t mix32(uint32_t h) {
  h ^= h >> 16;
  h *= 0x7FEB352Du;
  h ^= h >> 15;
  h *= 0x846CA68Bu;
  return h ^ (h >> 16);
}

// The bits whose upper ones are the e4m3 code of x / 2^e by stochastic rounding, |x / 2^e| <
// 256, lift = -120 - e: with 2^-120, e4m3's smallest normal 2^-6 becomes fp32's, so that the
// exponent and the upper three mantissa bits are the code, subnormal ones included, and the
// denormal product rounds where 2^-6 + |x / 2^e| would.  16 random bits (HIGH: the upper ones
// of u) are added to the 20 bits that the code drops, aligned with the highest of them.
template <bool HIGH>
__device__ __forceinline__ uint32_t encode(float x, int lift, uint32_t u) {
  const uint32_t t = __float_as_uint(__builtin_amdgcn_ldexpf(x, lift));
  uint32_t r;
  if (HIGH)
    asm("v_mad_u32_u16 %0, %1, 16, %2 op_sel:[1,0,0,0]" : "=v"(r) : "v"(u), "v"(t));
  else
    asm("v_mad_u32_u16 %0, %1, 16, %2" : "=v"(r) : "v"(u), "v"(t));
  return r;
}

// sqrt rounded to nearest for v = 0 and v >= 2^-100 (but for one v in 2^21, off by its last
// bit): the reciprocal root's product, corrected once by its exact residual.  11 operations
// where sqrtf, which scales small v, takes 18
__device__ __forceinline__ float root_of(float v) {
  const float y = __builtin_amdgcn_rsqf(fmaxf(v, 0x1p-100f));
  const float s = v * y;
  return fmaf(fmaf(-s, s, v), 0.5f * y, s);
}

// the scale 2^e of a block whose largest finite magnitude is a: a / 2^e in [128, 256)
__device__ __forceinline__ float scale_of(uint32_t bits) {
  const int e = int(bits >> 23) - 7;
  return __uint_as_float(uint32_t(e < 27 ? 27 : e) << 23);  // 2^-100 at least
}
// encode's lift for it
__device__ __forceinline__ int lift_of(float scale) { return 7 - int(__float_as_uint(scale) >> 23); }

// a b + c d, each product rounded: where they cancel the sum is 0, not a product's rounding
__device__ __forceinline__ double two_products(double a, double b, double c, double d) {
#pragma clang fp contract(off)
  return a * b + c * d;
}

// the bits of |x|, 0 where x is not finite
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t a = __float_as_uint(x) & 0x7FFFFFFFu;
  return a < kInfBits ? a : 0u;
}

// max over the 32 lanes that share a state block, in each of them, of bits that order as they
// are: rotations within the rows of 16, then the other row
template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
  const uint32_t o = uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 0xF, 0xF, false));
  return max(v, o);
}
__device__ __forceinline__ uint32_t max32(uint32_t v) {
  v = max_dpp<0x128>(v);  // row_ror 8, 4, 2, 1
  v = max_dpp<0x124>(v);
  v = max_dpp<0x122>(v);
  v = max_dpp<0x121>(v);
  return max(v, uint32_t(__shfl_xor(int(v), 16)));
}

// where a thread's elements of a chunk are
template <typename T>
struct Place {
  int tensor;
  int64_t left, e;  // elements from its first on (positive: some); the first one in the states
  T* p;
  const T* g;
  bool whole;       // all kPer, at 16-byte addresses
};

// what it reads of them
template <typename T, int BITS>
struct Loaded {
  T p[kPer], g[kPer];
  float m[kPer], v[kPer];
};
template <typename T>
struct Loaded<T, 8> {
  T p[kPer], g[kPer];
  uint32_t m[2], v[2];
  float ms, vs;
};

template <int N, typename T>
__device__ __forceinline__ void copy_vec(T* to, const T* from) {
  constexpr int kV = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
#pragma unroll
  for (int j = 0; j < N; j += kV)
    *reinterpret_cast<Pack<T, kV>*>(to + j) = *reinterpret_cast<const Pack<T, kV>*>(from + j);
}

template <typename T, int BITS>
__device__ __forceinline__ void load(const AdamArgs& a, const Place<T>& w, Loaded<T, BITS>& x) {
  if (w.whole) {
    copy_vec<kPer>(x.p, static_cast<const T*>(w.p));
    copy_vec<kPer>(x.g, w.g);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      x.p[j] = j < w.left ? w.p[j] : T(0.f);
      x.g[j] = j < w.left ? w.g[j] : T(0.f);
    }
  }
  if constexpr (BITS == 32) {
    const float* mp = static_cast<const float*>(a.m) + w.e;
    const float* vp = static_cast<const float*>(a.v) + w.e;
    if (w.left >= kPer) {
      copy_vec<kPer>(x.m, mp);
      copy_vec<kPer>(x.v, vp);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        x.m[j] = j < w.left ? mp[j] : 0.f;
        x.v[j] = j < w.left ? vp[j] : 0.f;
      }
    }
  } else {
    const uint8_t* mp = static_cast<const uint8_t*>(a.m) + w.e;
    const uint8_t* vp = static_cast<const uint8_t*>(a.v) + w.e;
    x.ms = x.vs = 0.f;
    if (w.left > 0) {
      x.ms = a.ms[w.e / kStateBlock];
      x.vs = a.vs[w.e / kStateBlock];
    }
    if (w.left >= kPer) {
      copy_vec<2>(x.m, reinterpret_cast<const uint32_t*>(mp));
      copy_vec<2>(x.v, reinterpret_cast<const uint32_t*>(vp));
    } else {
      x.m[0] = x.m[1] = x.v[0] = x.v[1] = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (j < w.left) {
          x.m[j / 4] |= uint32_t(mp[j]) << 8 * (j & 3);
          x.v[j / 4] |= uint32_t(vp[j]) << 8 * (j & 3);
        }
      }
    }
  }
}

// DECAYED: the gradient has weight_decay times the parameter added
template <typename T, int BITS, bool DECAYED>
__global__ void __launch_bounds__(kThreads, BITS == 32 ? kWaves32 : kWaves8) k_adam(const AdamArgs a) {
  const int lane = threadIdx.x & 63;
  const uint32_t c0 = lane < a.n ? a.t[lane].chunk0 : ~0u;
  const uint32_t c1 = lane + 64 < a.n ? a.t[lane + 64].chunk0 : ~0u;
  const double lr = a.lr_dev ? double(*a.lr_dev) : a.lr;
  const float keep = a.decoupled ? float(1.0 - lr * a.wd) : 1.f;
  int was = -1;
  float rate = 0.f, unbias = 0.f;
  uint32_t key = 0;
  auto place = [&](uint32_t chunk) {
    Place<T> w;
    w.tensor = wave_uniform(__popcll(__ballot(c0 <= chunk)) + __popcll(__ballot(c1 <= chunk)) - 1);
    const AdamTensor& t = a.t[w.tensor];
    const int64_t at = int64_t(chunk - t.chunk0) * kChunk + threadIdx.x * kPer;
    w.left = t.numel - at;
    w.e = t.first + at;
    w.p = static_cast<T*>(t.p) + at;
    w.g = static_cast<const T*>(t.g) + at;
    w.whole = w.left >= kPer &&
              ((reinterpret_cast<uintptr_t>(w.p) | reinterpret_cast<uintptr_t>(w.g)) & 15) == 0;
    return w;
  };
  for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
    const Place<T> w = place(chunk);
    Loaded<T, BITS> x;
    load<T, BITS>(a, w, x);
    if (w.tensor != was) {
      was = w.tensor;
      const uint32_t now = uint32_t(a.step[a.t[was].slot]) + 1u;
      rate = float(lr / (1.0 - power(a.b1, now)));
      unbias = float(1.0 / sqrt(1.0 - power(a.b2, now)));
      key = mix32(mix32(now) + a.seed);
    }
    const int64_t left = w.left, e = w.e;
    float p[kPer], g[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      p[j] = to_f32(x.p[j]);
      g[j] = to_f32(x.g[j]);
    }
    if constexpr (BITS == 32) {
      float* mp = static_cast<float*>(a.m) + e;
      float* vp = static_cast<float*>(a.v) + e;
      const float b1 = float(a.b1), b2 = float(a.b2), d1 = float(1.0 - a.b1), d2 = float(1.0 - a.b2);
      float (&m)[kPer] = x.m, (&v)[kPer] = x.v;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const float gj = DECAYED ? g[j] + float(a.wd) * p[j] : g[j];
        m[j] = b1 * m[j] + d1 * gj;
        v[j] = b2 * v[j] + d2 * gj * gj;
        p[j] = p[j] * keep - rate * (m[j] / (sqrtf(v[j]) * unbias + a.eps));
      }
      if (left >= kPer) {
        copy_vec<kPer>(mp, static_cast<const float*>(m));
        copy_vec<kPer>(vp, static_cast<const float*>(v));
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
      uint32_t (&mc)[2] = x.m, (&vc)[2] = x.v;
      float ms = x.ms, vs = x.vs;
      float m[kPer], r[kPer];
      uint32_t mmax = 0, rmax = 0, tiny = ~0u;  // bits
      const double d1 = 1.0 - a.b1, d2 = 1.0 - a.b2;
      const double b1ms = a.b1 * double(ms), b2vs = a.b2 * (double(vs) * double(vs));
      auto decode = [](uint32_t w, int j) {  // (the byte index has to be a literal)
        switch (j & 3) {
          case 0: return __builtin_amdgcn_cvt_f32_fp8(int(w), 0);
          case 1: return __builtin_amdgcn_cvt_f32_fp8(int(w), 1);
          case 2: return __builtin_amdgcn_cvt_f32_fp8(int(w), 2);
          default: return __builtin_amdgcn_cvt_f32_fp8(int(w), 3);
        }
      };
      // fp64, so that a moment next to a border between two scales or codes falls on its side;
      // the scales are powers of two, so that they round nothing wherever they are multiplied
      auto gradient = [&](int j) {
        const double gj = double(g[j]);
        return DECAYED ? two_products(gj, 1.0, a.wd, double(p[j])) : gj;
      };
      auto second = [&](int j, double gj) {
        const float c = decode(vc[j / 4], j);
        return float(two_products(b2vs, double(c * c), d2, gj * gj));
      };
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const double gj = gradient(j);
        m[j] = float(two_products(b1ms, double(decode(mc[j / 4], j)), d1, gj));
        const float v = second(j, gj);
        r[j] = root_of(v);
        tiny = min(tiny, __float_as_uint(v) - 1u);
        mmax = max(mmax, __float_as_uint(m[j]) & 0x7FFFFFFFu);
        rmax = max(rmax, __float_as_uint(r[j]));
      }
      bool special = (mmax > rmax ? mmax : rmax) >= kInfBits;
      if (special || tiny < 0x0D7FFFFFu) {  // 0 < v < 2^-100, or one that is not finite: sqrtf
        mmax = rmax = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          r[j] = sqrtf(second(j, gradient(j)));
          mmax = max(mmax, finite_bits(m[j]));  // the scales go by the finite ones
          rmax = max(rmax, finite_bits(r[j]));
        }
      }
      // (v_rcp_f32 is within 2^-23: two roundings, of an update whose moments are known to 2^-4)
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        p[j] = fmaf(p[j], keep, -rate * (m[j] * __builtin_amdgcn_rcpf(fmaf(r[j], unbias, a.eps))));
      ms = scale_of(max32(mmax));
      vs = scale_of(max32(rmax));
      const int ml = lift_of(ms), vl = lift_of(vs);
      const uint32_t k2 = (e >> 32) ? key ^ mix32(uint32_t(e >> 32)) : key;
      uint32_t me[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const uint32_t u = mix32(uint32_t(e + j) * 0x9E3779B1u + k2);
        const uint32_t w = encode<false>(m[j], ml, u);
        me[j] = (w << 4 & 0x7FFFFFFFu) | (w & 0x80000000u);  // sign and code: the upper byte
        // a root that is not 0 has no code 0
        const uint32_t c = max(encode<true>(r[j], vl, u) >> 20, min(__float_as_uint(r[j]), 1u));
        vc[j / 4] = (j & 3) ? vc[j / 4] | c << 8 * (j & 3) : c;
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)  // the upper bytes of four
        mc[k] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(me[4 * k + 3], me[4 * k + 2], 0x07030000u),
                                      __builtin_amdgcn_perm(me[4 * k + 1], me[4 * k], 0x00000703u),
                                      0x07060100u);
      if (special) {  // NaN and infinity: the NaN code
        for (int j = 0; j < kPer; ++j) {
          const uint32_t b = 0xFFu << 8 * (j & 3), nan = 0x7Fu << 8 * (j & 3);
          if ((__float_as_uint(m[j]) & 0x7FFFFFFFu) >= kInfBits) mc[j / 4] = (mc[j / 4] & ~b) | nan;
          if ((__float_as_uint(r[j]) & 0x7FFFFFFFu) >= kInfBits) vc[j / 4] = (vc[j / 4] & ~b) | nan;
        }
      }
      if (left >= kPer) {
        copy_vec<2>(reinterpret_cast<uint32_t*>(mp), static_cast<const uint32_t*>(mc));
        copy_vec<2>(reinterpret_cast<uint32_t*>(vp), static_cast<const uint32_t*>(vc));
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
#pragma unroll
    for (int j = 0; j < kPer; ++j) x.p[j] = from_f32<T>(p[j]);
    if (w.whole) {
      copy_vec<kPer>(w.p, static_cast<const T*>(x.p));
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (j < left) w.p[j] = x.p[j];
    }
  }
  // every block has read the step counts it needs: the last one here advances them
  __shared__ uint32_t last;
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t leaf = blockIdx.x % kLeaves;
    const uint32_t leaves = gridDim.x < kLeaves ? gridDim.x : kLeaves;
    const uint32_t here = (gridDim.x - leaf + kLeaves - 1) / kLeaves;  // blocks of this leaf
    last = 0u;
    if (atomicAdd(a.ticket + leaf * kLine, 1u) == here - 1) {
      a.ticket[leaf * kLine] = 0u;
      if (atomicAdd(a.ticket + kLeaves * kLine, 1u) == leaves - 1) {
        a.ticket[kLeaves * kLine] = 0u;
        last = 1u;
      }
    }
  }
  __syncthreads();
  if (last)
    for (int i = threadIdx.x; i < a.n; i += kThreads) a.step[a.t[i].slot] += 1;
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
    const int most = state_bits == 32 ? kMaxBlocks32 : kMaxBlocks8;
    const int grid = int(chunks < 1 ? 1 : chunks < most ? chunks : most);
    const gfd_status st = with_dtype(dtype, [&](auto tag) {
      using T = decltype(tag);
      const bool decayed = !decoupled && weight_decay != 0.0;
      if (state_bits == 32 && decayed)
        k_adam<T, 32, true><<<grid, kThreads, 0, stream>>>(a);
      else if (state_bits == 32)
        k_adam<T, 32, false><<<grid, kThreads, 0, stream>>>(a);
      else if (decayed)
        k_adam<T, 8, true><<<grid, kThreads, 0, stream>>>(a);
      else
        k_adam<T, 8, false><<<grid, kThreads, 0, stream>>>(a);
      GFD_LAUNCH_CHECK();
      return GFD_OK;
    });
    if (st != GFD_OK) return st;
  }
  return GFD_OK;
}

}  // extern "C"
