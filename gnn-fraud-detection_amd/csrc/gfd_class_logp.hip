// gfd_class_logp.hip -- log probabilities of given classes, entropy and the top
// alternatives of a classification head's logits, forward and backward.
//
//   lse = R + log S,  S = sum e^(x - R),  T = sum e^(x - R) (x - R)
//   log p_c = x_c - lse,  entropy = log S - T / S
//   dL/dx_c = -p_c (G + gH (log p_c + entropy)) + [c = t] g + sum_j [c = top_j] g_j
//
// Bound by memory: the forward reads every logit once, the backward reads it
// again and writes its gradient.  16-bit logits leave about 14 vector
// operations for an element at the card's copy rate, and the sums take ten (an
// exponential counts four), so the loop is kept to them:
//   * R is, while a row is read, any reference not far below its largest logit: a
//     lane moves its own only when a logit exceeds it by more than kSlack.  A
//     running maximum would be moved by one of the 64 lanes in nearly every
//     iteration.  The lanes' sums are joined about the largest logit.
//   * The top list is a wave's: entry j in lane j.  A vector of logits enters the
//     search only where its largest is above the list's last entry, the same
//     comparison as the reference's; the waves that share a row tell each other
//     their lists' last entries.
// Rows of up to kNarrow classes are read by teams of 1 to 32 lanes, longer ones
// by a wave, long ones by a block; few long rows are split over blocks whose
// partial results a second kernel joins.  2048 rows of 203769 bf16 logits: 153 to
// 161 us without a list (5.2 to 5.4 TB/s), 190 to 201 us with the best 8; backward
// 305 to 322 us.
#include "gfd_rowops.h"

using namespace gfd;

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
// classes of the team kernel: 32 lanes of 4 (100000 rows of 128 in bf16, no list and the best 5:
// 16 and 59 us, by a wave each 37 and 106; of 256 in teams of 64 lanes 38 and 124, by a wave 38
// and 104)
constexpr int kNarrow = 128;
constexpr int kMaxTop = 64;        // a list entry a lane
// classes of a split, at least (a row of 16384, the best 8: 17.5 us, of splits of 16384 19.4; a
// row of 1000000: 33 us, of splits of 2048 42)
constexpr int kMinSplit = 4096;
// rows are split below it (900 rows of 65536, the best 8: 56 us whole, 63 us in two)
constexpr int kFill = 512;
constexpr float kSlack = 8.f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();

__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// max that does not pass its operands through a canonicalisation first
__device__ __forceinline__ float max_f(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ float max3_f(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// reductions over the wave, uniform: lane 15 of a row of 16 collects its row's, rows 1 and 3
// the row before, rows 2 and 3 the first two; lanes without a source read ``none``
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float none, float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), CTRL, ROWS, 0xF, false));
}
template <typename F>
__device__ __forceinline__ float wave_reduce(float none, float v, F f) {
  v = f(v, dpp<0x111, 0xF>(none, v));  // row_shr 1, 2, 4, 8
  v = f(v, dpp<0x112, 0xF>(none, v));
  v = f(v, dpp<0x114, 0xF>(none, v));
  v = f(v, dpp<0x118, 0xF>(none, v));
  v = f(v, dpp<0x142, 0xA>(none, v));  // row_bcast 15, 31
  v = f(v, dpp<0x143, 0xC>(none, v));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
// the largest that is not NaN
__device__ __forceinline__ float wave_max(float v) {
  return wave_reduce(-kInf, v, [](float a, float b) { return max_f(a, b); });
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_reduce(0.f, v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float lane_of(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
template <int W>
__device__ __forceinline__ float team_sum(float v) {
#pragma unroll
  for (int d = 1; d < W; d <<= 1) v += __shfl_xor(v, d, W);
  return v;
}

// running sums about a reference
struct Sums {
  float r = -kInf, s = 0.f, t = 0.f;
  __device__ __forceinline__ void move(float to) {
    const bool none = r == -kInf;
    const float d = none ? 0.f : max_f(r - to, -1000.f);  // finite: e^d is 0 long before
    const float f = none ? 0.f : exp_of(d);
    t = f * (t + d * s);
    s *= f;
    r = to;
  }
  __device__ __forceinline__ void add(float x) { add_about(x, r == -kInf ? 0.f : r); }
  __device__ __forceinline__ void add_about(float x, float about) {
    const float d = x - about;
    const float e = exp_of(d);
    s += e;
    t = fmaf(e, max_f(d, -1000.f), t);  // e = 0 at d = -inf: adds 0
  }
  // the wave's sums about its largest logit, in every lane of it; ``most``: the lane's
  __device__ __forceinline__ void join(float most) {
    const float to = wave_max(most);
    if (to != -kInf) move(to);
    s = wave_sum(s);
    t = wave_sum(t);
  }
};

// a wave's list of the largest logits so far, larger first, equal ones by the
// lower class; entry j in lane j, lanes from ``size`` on NaN
__device__ __forceinline__ float above(float v) {  // the next float
  const uint32_t b = __float_as_uint(v);
  return __uint_as_float(v == 0.f ? 1u : v > 0.f ? b + 1 : b - 1);
}
__device__ __forceinline__ float below(float v) { return -above(-v); }

struct Entry {  // of a list
  float val;
  int cls;
};

// appends the wanted entries of the lanes to those found, up to kWave
__device__ __forceinline__ void gather(bool wanted, Entry e, Entry* found, int& count) {
  const unsigned long long some = __ballot(wanted);
  const int at = count + __builtin_amdgcn_mbcnt_hi(uint32_t(some >> 32),
                                                   __builtin_amdgcn_mbcnt_lo(uint32_t(some), 0u));
  if (wanted && at < kWave) found[at] = e;
  count += __popcll(some);
}

// a lane's entry's place among the ``count`` of the first lanes; behind them, a place of its own
__device__ __forceinline__ int rank_of(Entry e, int count) {
  const int lane = threadIdx.x & 63;
  int rank = lane < count ? 0 : lane;
  for (int i = 0; i < count; ++i) {
    const float v = lane_of(e.val, i);
    const int c = __builtin_amdgcn_readlane(e.cls, i);
    if (v > e.val || (v == e.val && c < e.cls)) ++rank;
  }
  return rank;
}

struct Top {
  float val = __builtin_nanf("");
  int cls = 0;
  int size = 0;                     // uniform
  float floor = -kInf;              // of a full list, uniform: its last entry
  int floor_cls = INT32_MAX;

  __device__ __forceinline__ void put(float v, int c, int top) {
    const int lane = threadIdx.x & 63;
    const int at = __popcll(__ballot(val > v || (val == v && cls < c)));
    // wave_shr 1: the entry of the lane before
    const float up = dpp<0x138, 0xF>(val, val);
    const int up_c = __builtin_amdgcn_update_dpp(cls, cls, 0x138, 0xF, 0xF, false);
    val = lane > at ? up : lane == at ? v : val;
    cls = lane > at ? up_c : lane == at ? c : cls;
    val = lane < top ? val : __builtin_nanf("");
    size = size < top ? size + 1 : top;
    if (size == top) {
      floor = lane_of(val, top - 1);
      floor_cls = __builtin_amdgcn_readlane(cls, top - 1);
    }
  }

  // A bound from below of the ``top``-th largest of the lanes' values (NaN: none), of which
  // about that many are not below it: the upper half of its bits, found one by one
  __device__ __forceinline__ static float bound_of(float v, int top) {
    if (__popcll(__ballot(v == v)) < top) return -kInf;
    const uint32_t b = __float_as_uint(v + 0.f);
    // unsigned bits that order like the values
    const uint32_t u = v == v ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
    uint32_t low = 0;
#pragma unroll 1
    for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1) {
      const int many = __popcll(__ballot(u >= (low | bit)));
      if (many >= top) low |= bit;
      if (many == top) break;
    }
    if (low < 0x00800000u) return -kInf;  // -inf, or what would be a NaN's bits
    return __uint_as_float(low & 0x80000000u ? low & 0x7FFFFFFFu : ~low);
  }

  // would a candidate enter the list
  __device__ __forceinline__ bool fits(float v, int c, int top) const {
    return size < top ? v == v : v > floor || (v == floor && c < floor_cls);
  }

  // a candidate a lane; ``some``: the lanes that have one that fits
  __device__ __forceinline__ void merge(unsigned long long some, float v, int c, int top) {
    while (some) {
      const int l = __ffsll(some) - 1;
      put(lane_of(v, l), __builtin_amdgcn_readlane(c, l), top);
      some &= some - 1;
      if (size == top) some &= __ballot(fits(v, c, top));
    }
  }

  // a listed entry a lane, NaN: none
  __device__ __forceinline__ void join(float v, int c, int top) {
    const float low = size < top ? bound_of(v, top) : -kInf;
    merge(__ballot(v >= low && fits(v, c, top)), v, c, top);
  }

  // The logits x of a wave's vector, ``have`` of a lane's N from class cls0 on, those below
  // ``least`` not wanted.  They come in the order of their classes, lane by lane, and (ORDERED)
  // after all lower classes: once the list is full, one that equals its last entry is not.
  // (Many at once by their ranks, as k_fwd_join does, is no faster: 20000 rows of 16384, the best
  // 5: 172 us, one by one 159; a row of 203769, the best 10: 19 and 20 us.)
  template <bool ORDERED, int N>
  __device__ __forceinline__ void take(const float (&x)[N], int have, int cls0, int top, float least) {
    float best = __builtin_nanf("");
#pragma unroll
    for (int j = 0; j < N; ++j) best = max_f(best, j < have ? x[j] : __builtin_nanf(""));
    float low = size < top ? bound_of(best, top) : ORDERED ? above(floor) : floor;
    low = max_f(low, least);
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) bits |= x[j] >= low ? 1u << j : 0u;
    bits &= (1u << have) - 1;
    unsigned long long some = __ballot(bits != 0);
    while (some) {
      const int l = __ffsll(some) - 1;
      uint32_t b = __builtin_amdgcn_readlane(bits, l);
      const int c0 = __builtin_amdgcn_readlane(cls0, l);
      for (; b; b &= b - 1) {
        const int j = __ffs(b) - 1;
        float v = x[0];
#pragma unroll
        for (int i = 1; i < N; ++i) v = i == j ? x[i] : v;
        const float m = lane_of(v, l);
        if (size < top || m > floor || (!ORDERED && m == floor && c0 + j < floor_cls)) put(m, c0 + j, top);
      }
      some &= some - 1;
      if (size == top) some &= __ballot(ORDERED ? best > floor : best >= floor);
    }
  }
};

struct RowOut {
  const int64_t* target;
  int64_t ignore;
  float* logp;
  float* entropy;
  float* top_logp;
  int64_t* top_class;
  float* stats;
};

// log p of a logit from the row's statistics (R, log S); an empty row: -inf
__device__ __forceinline__ float logp_of(float x, float r, float ls) {
  return r == -kInf && ls == -kInf ? -kInf : (x - r) - ls;
}

// the given class of a row and its logit
struct Given {
  int64_t c;
  float x;
  bool known;  // in the classes
};
template <typename T>
__device__ __forceinline__ Given given_of(const RowOut& o, int64_t row, const T* x, int64_t classes) {
  Given g = {0, 0.f, false};
  if (o.logp) {
    g.c = o.target[row];
    g.known = g.c >= 0 && g.c < classes;
    if (g.known) g.x = to_f32(x[g.c]);
  }
  return g;
}

__device__ __forceinline__ void write_row(const RowOut& o, int64_t row, const Given& g, float r, float s,
                                          float t) {
  const float ls = s == 0.f ? -kInf : logf(s);
  o.stats[2 * row] = r;
  o.stats[2 * row + 1] = ls;
  o.entropy[row] = s == 0.f ? 0.f : ls - t / s;
  if (o.logp)
    o.logp[row] = g.c == o.ignore ? 0.f : g.known ? logp_of(g.x, r, ls) : __builtin_nanf("");
}

// ---------------------------------------------------------------------------
// up to 128 classes: a team of W lanes a row, 4 classes a lane (class j * W + l)
// ---------------------------------------------------------------------------
template <typename T, int W>
__global__ void __launch_bounds__(kThreads) k_fwd_narrow(const T* __restrict__ x, int64_t rows,
                                                         int classes, int64_t stride, int top,
                                                         RowOut o) {
  const int l = threadIdx.x & (W - 1);
  const int64_t teams = int64_t(gridDim.x) * (kThreads / W);
  const int64_t first = int64_t(blockIdx.x) * (kThreads / W) + threadIdx.x / W;
  for (int64_t row = first; row < rows; row += teams) {
    const T* xr = x + row * stride;
    float v[4];
    Sums a;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = j * W + l < classes ? to_f32(xr[j * W + l]) : -kInf;
      a.r = max_f(a.r, v[j]);
    }
#pragma unroll
    for (int d = 1; d < W; d <<= 1) a.r = max_f(a.r, __shfl_xor(a.r, d, W));
#pragma unroll
    for (int j = 0; j < 4; ++j) a.add(v[j]);
    a.s = team_sum<W>(a.s);
    a.t = team_sum<W>(a.t);
    if (l == 0) write_row(o, row, given_of(o, row, xr, classes), a.r, a.s, a.t);
    if (top) {
      const float ls = a.s == 0.f ? -kInf : logf(a.s);
      // a taken entry, one outside of the classes and NaN are none: NaN
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j * W + l >= classes) v[j] = __builtin_nanf("");
      for (int n = 0; n < top; ++n) {
        float bv = __builtin_nanf("");
        int bc = INT32_MAX;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (v[j] > bv || (bv != bv && v[j] == v[j])) {
            bv = v[j];
            bc = j * W + l;
          }
        }
#pragma unroll
        for (int d = 1; d < W; d <<= 1) {
          const float ov = __shfl_xor(bv, d, W);
          const int oc = __shfl_xor(bc, d, W);
          if (ov > bv || (ov == bv && oc < bc) || (bv != bv && ov == ov)) {
            bv = ov;
            bc = oc;
          }
        }
        if (l == 0) {  // (of a row with a NaN some class: the first)
          o.top_class[row * top + n] = bv == bv ? bc : 0;
          o.top_logp[row * top + n] = logp_of(bv, a.r, ls);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (bc == j * W + l) v[j] = __builtin_nanf("");
      }
    }
  }
}

// ---------------------------------------------------------------------------
// more classes: W waves of a block a row, or a split of one
// ---------------------------------------------------------------------------
struct Partial {  // of a wave or a split
  float r, s, t;
};

// sums, largest logit and top list of the elements [begin, end) of a row that this wave reads:
// wave w of W.  best_floor (LDS, nullable): the highest floor of the waves' lists, a bound
// from below of the row's list
template <typename T, int W>
__device__ __forceinline__ void scan_row(const T* xr, int begin, int end, int w, int top, Sums& a,
                                         float& most, Top& best, volatile float* best_floor) {
  constexpr int V = 16 / sizeof(T);
  constexpr int U = 2;  // vectors in flight a lane
  const int lane = threadIdx.x & 63;
  float bound = -kInf;  // a vector whose largest logit is not above it needs no second look
  float least = -kInf;  // nor is one below this wanted in the list
  auto limit = [&]() {
    bound = a.r + kSlack;
    if (top) {
      // equal to another wave's floor: wanted, its class may be the lower one
      const float f = best.size < top ? -kInf : best.floor >= least ? best.floor : below(least);
      bound = f < bound ? f : bound;
    }
  };
  // [begin, lo) and [hi, end): what the 16-byte vectors leave, under 16 classes
  const int head = int((16 - (reinterpret_cast<uintptr_t>(xr + begin) & 15)) & 15) / int(sizeof(T));
  const int lo = begin + (head < end - begin ? head : end - begin);
  const int vecs = (end - lo) / V, hi = lo + vecs * V;
  const int rest = w == 0 ? lo - begin + end - hi : 0;
  const auto* p = reinterpret_cast<const Pack<T, V>*>(xr + lo);
  // groups of U vectors, then the rest as a group of its own
  for (int v0 = w * 64;; v0 += W * 64 * U) {
    const bool last = v0 >= vecs;
    if (last && rest <= 0) break;
    Pack<T, V> q[U];
    if (v0 + (U - 1) * W * 64 + 64 <= vecs) {
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = p[v0 + u * W * 64 + lane];
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) q[u].v[j] = from_f32<T>(-kInf);
      if (!last) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (v0 + u * W * 64 + lane < vecs) q[u] = p[v0 + u * W * 64 + lane];
      } else if (lane < rest) {  // one element a lane, those before the vectors first
        q[0].v[0] = xr[lane < lo - begin ? begin + lane : hi + lane - (lo - begin)];
      }
    }
    // vectors of this group that some lane has
    const int live = last ? 1 : min(U, (vecs - v0 + W * 64 - 1) / (W * 64));
    if (W > 1 && top) {
      const float f = *best_floor;
      if (__ballot(f > least)) {
        least = f;
        limit();
      }
    }
    float m[U], all = -kInf;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] = -kInf;
#pragma unroll
      for (int j = 0; j < V; j += 2) m[u] = max3_f(m[u], to_f32(q[u].v[j]), to_f32(q[u].v[j + 1]));
      all = max_f(all, m[u]);
    }
    most = max_f(most, all);
    if (__ballot(all > bound) || (top && (last || best.size < top))) {
      if (all > a.r + kSlack) a.move(all);
      if (top) {
        uint32_t todo = 0;  // the vectors with something for the list
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (u < live && (last || best.size < top || __ballot(m[u] > best.floor && m[u] >= least)))
            todo |= 1u << u;
#pragma unroll 1
        for (; todo; todo &= todo - 1) {
          const int u = __ffs(todo) - 1;
          Pack<T, V> c = q[0];
#pragma unroll
          for (int k = 1; k < U; ++k)
            if (u == k) c = q[k];
          float y[V];
#pragma unroll
          for (int j = 0; j < V; ++j) y[j] = to_f32(c.v[j]);
          if (!last) {
            const int v = v0 + u * W * 64 + lane;
            best.template take<true>(y, v < vecs ? V : 0, lo + v * V, top, least);
          } else {
            const float z[1] = {y[0]};
            best.template take<false>(z, lane < rest ? 1 : 0,
                                      lane < lo - begin ? begin + lane : hi + lane - (lo - begin), top, least);
          }
          if (W > 1 && best.size == top && best.floor > least) *best_floor = least = best.floor;
        }
      }
      limit();
    }
    const float r = a.r == -kInf ? 0.f : a.r;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u < live) {
#pragma unroll
        for (int j = 0; j < V; ++j) a.add_about(to_f32(q[u].v[j]), r);
      }
    }
    if (last) break;
  }
}

// the list of a row, a lane an entry; of a row with a NaN, some classes
__device__ __forceinline__ void write_top(const RowOut& o, int64_t row, int top, const Top& best,
                                          float r, float s) {
  const int lane = threadIdx.x & 63;
  if (lane < top) {
    const float ls = s == 0.f ? -kInf : logf(s);
    o.top_class[row * top + lane] = lane < best.size ? best.cls : 0;
    o.top_logp[row * top + lane] = logp_of(best.val, r, ls);
  }
}

// (8 waves a SIMD, 64 registers: with 4 vectors in flight and 5 waves, or the next group read
// ahead, the kernel is up to 15 % slower)
template <typename T, int W, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 8) k_fwd_wide(const T* __restrict__ x, int64_t rows,
                                                       int classes, int64_t stride, int top,
                                                       int splits, int per_split,
                                                       Partial* __restrict__ part,
                                                       Entry* __restrict__ part_top, RowOut o) {
  __shared__ Partial sums[kWaves];
  __shared__ Entry lists[W > 1 ? W * kMaxTop : 1];
  __shared__ float best_floor;
  const int lane = threadIdx.x & 63, wave = wave_uniform(threadIdx.x >> 6);
  const int64_t jobs = rows * (SPLIT ? splits : 1);
  const int64_t step = int64_t(gridDim.x) * (kWaves / W);
  // every wave of a block runs the same number of iterations (barriers inside)
  for (int64_t job0 = int64_t(blockIdx.x) * (kWaves / W); job0 < jobs; job0 += step) {
    const int64_t job = job0 + (W > 1 ? 0 : wave);
    if (W == 1 && job >= jobs) break;
    const int64_t row = SPLIT ? job / splits : job;
    const int begin = SPLIT ? int(job - row * splits) * per_split : 0;
    const int end = SPLIT ? (begin + per_split < classes ? begin + per_split : classes) : classes;
    const T* xr = x + row * stride;
    if (W > 1 && top) {
      if (threadIdx.x == 0) best_floor = -kInf;
      __syncthreads();
    }
    Sums a;
    Top best;
    float most = -kInf;
    scan_row<T, W>(xr, begin, end, W > 1 ? wave : 0, top, a, most, best, &best_floor);
    a.join(most);
    if (W > 1) {
      if (lane == 0) sums[wave] = {a.r, a.s, a.t};
      if (wave > 0 && lane < top) lists[wave * top + lane] = {best.val, best.cls};
      __syncthreads();
      if (wave == 0) {
        a = Sums();
        if (lane < W) {
          a.r = sums[lane].r;
          a.s = sums[lane].s;
          a.t = sums[lane].t;
        }
        a.join(a.r);
        if (top) {
          for (int w = 1; w < W; ++w) {
            Entry e = {__builtin_nanf(""), 0};
            if (lane < top) e = lists[w * top + lane];
            best.join(e.val, e.cls, top);
          }
        }
      }
    }
    if (W == 1 || wave == 0) {
      if (SPLIT) {
        if (lane == 0) part[job] = {a.r, a.s, a.t};
        if (lane < top) part_top[job * top + lane] = {best.val, best.cls};
      } else {
        if (lane == 0) write_row(o, row, given_of(o, row, xr, classes), a.r, a.s, a.t);
        write_top(o, row, top, best, a.r, a.s);
      }
    }
    if (W > 1) __syncthreads();  // the next row writes the lists
  }
}

// a wave a row: the splits' sums and lists.  ``need`` lanes whose lists' entry number ``level`` is
// not below some value have ``top`` entries that are not: a bound of the row's list.  The few
// entries not below it are gathered, and each counts those before it (one row of 203769, the
// best 10: 4.7 us; entries put into a list one by one 11.3 us)
template <typename T>
__global__ void __launch_bounds__(kWave) k_fwd_join(const T* __restrict__ x, int64_t rows,
                                                    int classes, int64_t stride, int top,
                                                    int splits, const Partial* __restrict__ part,
                                                    const Entry* __restrict__ part_top, RowOut o) {
  __shared__ Entry found[kWave];
  const int lane = threadIdx.x;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    // everything it reads, before anything waits for it
    const int n = splits * top;
    const Entry* from = part_top + row * n;
    const Given given = given_of(o, row, x + row * stride, classes);
    Partial p = {-kInf, 0.f, 0.f};
    const int lanes = splits < kWave ? splits : kWave;
    const int level = (top - 1) / lanes, need = (top + level) / (level + 1);
    float head = __builtin_nanf("");
    if (lane < splits) {
      p = part[row * splits + lane];
      if (top) head = from[lane * top + level].val;
    }
    Entry e[8];
    auto read = [&](int i0) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        e[k] = {__builtin_nanf(""), 0};
        if (i0 + k * 64 + lane < n) e[k] = from[i0 + k * 64 + lane];
      }
    };
    read(0);
    Sums a;
    for (int i = lane; i < splits;) {
      if (p.r > a.r) a.move(p.r);
      Sums b;
      b.r = p.r;
      b.s = p.s;
      b.t = p.t;
      if (p.r != -kInf) b.move(a.r);
      a.s += b.s;
      a.t += b.t;
      if ((i += 64) < splits) {
        p = part[row * splits + i];
        if (top) head = max_f(head, from[i * top + level].val);
      }
    }
    a.join(a.r);
    if (lane == 0) write_row(o, row, given, a.r, a.s, a.t);
    if (top) {
      const float least = Top::bound_of(head, need);
      int count = 0;  // of the entries not below it
      for (int i0 = 0; i0 < n;) {
#pragma unroll
        for (int k = 0; k < 8; ++k) gather(e[k].val >= least, e[k], found, count);
        if ((i0 += 512) < n) read(i0);
      }
      __syncthreads();
      if (count <= kWave) {
        Entry e = {__builtin_nanf(""), 0};
        if (lane < count) e = found[lane];
        const int rank = rank_of(e, count);
        if (rank < top) {
          o.top_class[row * top + rank] = e.cls;
          o.top_logp[row * top + rank] = logp_of(e.val, a.r, a.s == 0.f ? -kInf : logf(a.s));
        }
      } else {  // many equal ones
        Top best;
        for (int i = 0; i < n; i += 64) {
          Entry e = {__builtin_nanf(""), 0};
          if (i + lane < n) e = from[i + lane];
          best.join(e.val, e.cls, top);
        }
        write_top(o, row, top, best, a.r, a.s);
      }
      __syncthreads();  // the next row's entries
    }
  }
}

// A row by one wave, or by a block's: a wave where the rows fill the card, which costs no joins
// (2000 rows of 4096, the best 5: 19 us, by blocks 22; 20000 rows: 68 and 132), a block where
// they do not (256 rows: 17 and 12 us).  Longer rows read the same by either, but a list a wave
// is four lists a row (20000 rows of 16384, the best 5: 148 and 239 us; 4096 rows of 65536: 119
// and 123; no list: 116 and 109).
inline bool by_wave(int64_t rows, int64_t classes, int top) {
  return classes <= 1024 || (rows >= 1024 && classes <= 4096) ||
         (top > 0 && rows >= 4096 && classes <= 65536);
}

// how many blocks share a row, and the classes of one (a multiple of 16)
inline int splits_of(int64_t rows, int64_t classes, int top) {
  if (by_wave(rows, classes, top) || rows >= kFill) return 1;
  const int64_t by_rows = (kFill + rows - 1) / rows;
  const int64_t by_classes = (classes + kMinSplit - 1) / kMinSplit;
  return int(by_rows < by_classes ? by_rows : by_classes);
}
inline int per_split_of(int64_t classes, int splits) {
  return int(align_up(size_t((classes + splits - 1) / splits), 16));
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
struct BwdArgs {
  const int64_t* target;
  int64_t ignore;
  int top;
  const int64_t* top_class;
  const float* stats;
  const float* entropy;
  const float* g_logp;
  const float* g_entropy;
  const float* g_top;
};

struct BwdRow {
  float r, ls, given, total, bonus, ent;
  int64_t target;  // -1: none
  bool empty, bad;
};

__device__ __forceinline__ BwdRow bwd_row(const BwdArgs& b, int64_t row, int64_t classes) {
  BwdRow w;
  w.r = b.stats[2 * row];
  w.ls = b.stats[2 * row + 1];
  w.ent = b.entropy[row];
  w.empty = w.r == -kInf && w.ls == -kInf;
  w.given = 0.f;
  w.target = -1;
  w.bad = false;
  if (b.g_logp) {
    const int64_t c = b.target[row];
    if (c != b.ignore) {
      w.given = b.g_logp[row];
      w.target = c;
      w.bad = c < 0 || c >= classes;
    }
  }
  w.total = w.given;
  if (b.g_top)
    for (int j = 0; j < b.top; ++j) w.total += b.g_top[row * b.top + j];
  if (w.bad) w.total = __builtin_nanf("");
  w.bonus = b.g_entropy ? b.g_entropy[row] : 0.f;
  return w;
}

// the gradient apart from what the given and the listed classes add
__device__ __forceinline__ float bwd_dense(const BwdRow& w, float x) {
  const float lp = (x - w.r) - w.ls;
  const float p = exp_of(lp);
  return -p * (w.total + w.bonus * (max_f(lp, -1000.f) + w.ent));
}

// L lanes of a block a row, or a part of one; V elements an access (1: one element)
template <typename T, int V, int L>
__global__ void __launch_bounds__(kThreads) k_bwd(const T* __restrict__ x, int64_t rows,
                                                  int classes, int64_t stride, int parts,
                                                  int per_part, BwdArgs b, T* __restrict__ out) {
  const int lane = threadIdx.x % L;
  // (known to be uniform, a row's numbers come by scalar loads: 350 -> 320 us over 417M logits)
  const int team = L >= kThreads ? 0 : L >= kWave ? wave_uniform(threadIdx.x / L) : threadIdx.x / L;
  const int64_t jobs = rows * parts, step = int64_t(gridDim.x) * (kThreads / L);
  for (int64_t job = int64_t(blockIdx.x) * (kThreads / L) + team; job < jobs; job += step) {
    const int64_t row = parts == 1 ? job : job / parts;
    const int begin = int(job - row * parts) * per_part;
    const int end = begin + per_part < classes ? begin + per_part : classes;
    const BwdRow w = bwd_row(b, row, classes);
    const T* xr = x + row * stride;
    T* gr = out + row * classes;
    auto extra = [&](int c) {  // what the given and the listed classes add at class c
      float g = c == w.target ? w.given : 0.f;
      if (b.g_top)
        for (int j = 0; j < b.top; ++j)
          if (b.top_class[row * b.top + j] == c) g += b.g_top[row * b.top + j];
      return g;
    };
    auto at = [&](int c) {
      gr[c] = from_f32<T>(w.empty ? 0.f : bwd_dense(w, to_f32(xr[c])) + extra(c));
    };
    int lo = begin, vecs = 0;
    if (V > 1) {
      const int head = int((16 - (reinterpret_cast<uintptr_t>(xr + begin) & 15)) & 15) / int(sizeof(T));
      lo = begin + (head < end - begin ? head : end - begin);
      vecs = (end - lo) / V;
      const auto* px = reinterpret_cast<const Pack<T, V>*>(xr + lo);
      auto* pg = reinterpret_cast<Pack<T, V>*>(gr + lo);
      for (int v = lane; v < vecs; v += L) {
        const Pack<T, V> q = px[v];
        const int c0 = lo + v * V;
        float g[V];
#pragma unroll
        for (int j = 0; j < V; ++j) g[j] = w.empty ? 0.f : bwd_dense(w, to_f32(q.v[j]));
        if (!w.empty) {
          if (w.target >= c0 && w.target < c0 + V) {
#pragma unroll
            for (int j = 0; j < V; ++j) g[j] += c0 + j == w.target ? w.given : 0.f;
          }
          if (b.g_top) {
            for (int i = 0; i < b.top; ++i) {
              const int64_t c = b.top_class[row * b.top + i];
              if (c >= c0 && c < c0 + V) {
#pragma unroll
                for (int j = 0; j < V; ++j) g[j] += c0 + j == c ? b.g_top[row * b.top + i] : 0.f;
              }
            }
          }
        }
        Pack<T, V> r;
#pragma unroll
        for (int j = 0; j < V; ++j) r.v[j] = from_f32<T>(g[j]);
        pg[v] = r;
      }
    }
    // what the vectors leave, or everything
    const int before = lo - begin, tail = lo + vecs * V;
    for (int i = lane; i < before + end - tail; i += L) at(i < before ? begin + i : tail + i - before);
  }
}

inline bool bad_shape(int64_t rows, int64_t classes, int64_t stride, int top) {
  return rows < 0 || classes < 1 || classes >= (int64_t(1) << 31) - 65536 || top < 0 ||
         top > kMaxTop || top > classes || (rows > 1 && stride < 0) ||
         rows > (int64_t(1) << 40);
}

}  // namespace

extern "C" {

size_t gfd_class_logp_workspace_size(int64_t rows, int64_t classes, int top) {
  if (bad_shape(rows, classes, 0, top) || rows == 0) return 0;
  const int s = splits_of(rows, classes, top);
  if (s == 1) return 0;
  Sizer z;
  z.take<Partial>(size_t(rows) * s);
  z.take<Entry>(size_t(rows) * s * top);
  return z.off;
}

gfd_status gfd_class_logp_fwd(const void* logits, int dtype, int64_t rows, int64_t classes,
                              int64_t row_stride, const int64_t* target, int64_t ignore_index,
                              int top, float* logp, float* entropy, float* top_logp,
                              int64_t* top_class, float* stats, void* ws, size_t ws_bytes,
                              gfd_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (!float_dtype(dtype) || bad_shape(rows, classes, row_stride, top)) return GFD_ERR_ARGUMENT;
  if (rows == 0) return GFD_OK;
  if (!logits || !entropy || !stats || (logp && !target) || (top && (!top_logp || !top_class)))
    return GFD_ERR_ARGUMENT;
  if (!aligned_to(logits, dtype_size(dtype))) return GFD_ERR_ARGUMENT;
  const RowOut o{target, ignore_index, logp, entropy, top_logp, top_class, stats};
  const int n = int(classes);
  const int splits = splits_of(rows, classes, top);
  Partial* part = nullptr;
  Entry* part_top = nullptr;
  if (splits > 1) {
    Carve c(ws, ws_bytes);
    part = c.take<Partial>(size_t(rows) * splits);
    part_top = c.take<Entry>(size_t(rows) * splits * top);
    if (!c.ok) return GFD_ERR_WORKSPACE;
  }
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    const T* x = static_cast<const T*>(logits);
    auto narrow = [&](auto w) {
      constexpr int W = decltype(w)::value;
      const int64_t per = kThreads / W, blocks = (rows + per - 1) / per;
      k_fwd_narrow<T, W><<<int(blocks < 16384 ? blocks : 16384), kThreads, 0, stream>>>(
          x, rows, n, row_stride, top, o);
    };
    if (n <= 4) {
      narrow(std::integral_constant<int, 1>{});
    } else if (n <= 16) {
      narrow(std::integral_constant<int, 4>{});
    } else if (n <= 64) {
      narrow(std::integral_constant<int, 16>{});
    } else if (n <= kNarrow) {
      narrow(std::integral_constant<int, 32>{});
    } else if (by_wave(rows, classes, top)) {
      const int64_t blocks = (rows + kWaves - 1) / kWaves;
      k_fwd_wide<T, 1, false><<<int(blocks < 65536 ? blocks : 65536), kThreads, 0, stream>>>(
          x, rows, n, row_stride, top, 1, n, nullptr, nullptr, o);
    } else if (splits == 1) {
      k_fwd_wide<T, kWaves, false><<<int(rows < 65536 ? rows : 65536), kThreads, 0, stream>>>(
          x, rows, n, row_stride, top, 1, n, nullptr, nullptr, o);
    } else {
      k_fwd_wide<T, kWaves, true><<<int(rows * splits), kThreads, 0, stream>>>(
          x, rows, n, row_stride, top, splits, per_split_of(classes, splits), part, part_top, o);
      GFD_LAUNCH_CHECK();
      k_fwd_join<T><<<int(rows), kWave, 0, stream>>>(x, rows, n, row_stride, top, splits, part,
                                                     part_top, o);
    }
    GFD_LAUNCH_CHECK();
    return GFD_OK;
  });
}

gfd_status gfd_class_logp_bwd(const void* logits, int dtype, int64_t rows, int64_t classes,
                              int64_t row_stride, const int64_t* target, int64_t ignore_index,
                              int top, const int64_t* top_class, const float* stats,
                              const float* entropy, const float* grad_logp,
                              const float* grad_entropy, const float* grad_top,
                              void* grad_logits, gfd_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (!float_dtype(dtype) || bad_shape(rows, classes, row_stride, top)) return GFD_ERR_ARGUMENT;
  if (rows == 0) return GFD_OK;
  if (!logits || !stats || !entropy || !grad_logits || (grad_logp && !target) ||
      (grad_top && top && !top_class))
    return GFD_ERR_ARGUMENT;
  if (!aligned_to(logits, dtype_size(dtype)) || !aligned_to(grad_logits, dtype_size(dtype)))
    return GFD_ERR_ARGUMENT;
  const BwdArgs b{target, ignore_index, top, top_class, stats, entropy, grad_logp, grad_entropy,
                  top ? grad_top : nullptr};
  const int n = int(classes);
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    constexpr int V = 16 / sizeof(T);
    const T* x = static_cast<const T*>(logits);
    T* g = static_cast<T*>(grad_logits);
    auto launch = [&](auto v, auto l, int parts, int per) {
      constexpr int VV = decltype(v)::value, L = decltype(l)::value;
      const int64_t blocks = (rows * parts + kThreads / L - 1) / (kThreads / L);
      k_bwd<T, VV, L><<<int(blocks < 65536 ? blocks : 65536), kThreads, 0, stream>>>(
          x, rows, n, row_stride, parts, per, b, g);
    };
    using std::integral_constant;
    const integral_constant<int, 1> one;
    const integral_constant<int, V> vec;
    // 16-byte vectors where every row of both starts at the same place of one
    const bool same = (reinterpret_cast<uintptr_t>(x) - reinterpret_cast<uintptr_t>(g)) % 16 == 0 &&
                      (rows == 1 || (row_stride - classes) * int64_t(sizeof(T)) % 16 == 0);
    // 16 lanes up to 512 classes: 100000 rows of 256 23 us, of 512 36 us, a wave a row 44 and 50 us
    // (1000 rows 4.5 and 5.7 us, a wave 4.0); 256 rows of 4096: a wave a row 7.8 us, a block 4.6 us
    if (n <= 4) {
      launch(one, integral_constant<int, 1>{}, 1, n);
    } else if (n <= 16) {
      launch(one, integral_constant<int, 4>{}, 1, n);
    } else if (n <= 128) {
      launch(one, integral_constant<int, 16>{}, 1, n);
    } else if (n <= 512 && same) {
      launch(vec, integral_constant<int, 16>{}, 1, n);
    } else if (by_wave(rows, classes, 0)) {
      if (same) launch(vec, integral_constant<int, 64>{}, 1, n);
      else launch(one, integral_constant<int, 64>{}, 1, n);
    } else {
      const int parts = (n + 8191) / 8192, per = int(align_up(size_t((n + parts - 1) / parts), 16));
      if (same) launch(vec, integral_constant<int, 256>{}, parts, per);
      else launch(one, integral_constant<int, 256>{}, parts, per);
    }
    GFD_LAUNCH_CHECK();
    return GFD_OK;
  });
}

}  // extern "C"
