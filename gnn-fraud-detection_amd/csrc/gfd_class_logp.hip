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
//   * R is any reference not far below the row's largest logit, not that logit:
//     a lane moves its own only when a logit exceeds it by more than kSlack.  A
//     running maximum would be moved by one of the 64 lanes in nearly every
//     iteration.
//   * The top list is a wave's: entry j in lane j.  A vector of logits enters the
//     search only where its largest is above the list's last entry, the same
//     comparison as the reference's.
// Rows of up to kNarrow classes are read by teams of 1 to 32 lanes, longer ones
// by a wave, long ones by a block; few long rows are split over blocks whose
// partial results a second kernel joins.
#include "gfd_rowops.h"

using namespace gfd;

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kNarrow = 128;       // classes of the team kernel: 32 lanes of 4
constexpr int kWaveRow = 4096;     // classes a single wave reads
constexpr int kMaxTop = 64;        // a list entry a lane
constexpr int kMinSplit = 4096;    // classes of a split, at least
constexpr int kFill = 1024;        // blocks that fill the card: rows are split below it
constexpr float kSlack = 8.f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_inff();
constexpr int kNone = INT32_MIN;   // below the key of every logit

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

// int32 that orders like the logit; -0 as +0, NaN as -inf
__device__ __forceinline__ int key_of(float x) {
  x = x == x ? x + 0.f : -kInf;
  const int b = __float_as_int(x);
  return b < 0 ? b ^ 0x7FFFFFFF : b;
}
__device__ __forceinline__ float value_of(int key) {
  return __int_as_float(key < 0 ? key ^ 0x7FFFFFFF : key);
}

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_max(int v) {
  const int o = __builtin_amdgcn_update_dpp(kNone, v, CTRL, ROWS, 0xF, false);
  return v > o ? v : o;
}
// max over the wave, in every lane
__device__ __forceinline__ int wave_max(int v) {
  v = dpp_max<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8: lane 15 of a row holds its row's
  v = dpp_max<0x112, 0xF>(v);
  v = dpp_max<0x114, 0xF>(v);
  v = dpp_max<0x118, 0xF>(v);
  v = dpp_max<0x142, 0xA>(v);  // row_bcast 15 into rows 1 and 3
  v = dpp_max<0x143, 0xC>(v);  // row_bcast 31 into rows 2 and 3
  return __builtin_amdgcn_readlane(v, 63);
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
  __device__ __forceinline__ void add(float x) {
    const float d = x - (r == -kInf ? 0.f : r);
    const float e = exp_of(d);
    s += e;
    t = fmaf(e, max_f(d, -1000.f), t);  // e = 0 at d = -inf: adds 0
  }
  // the team's sums, in every lane of it
  template <int W>
  __device__ __forceinline__ void join() {
    float to = r;
#pragma unroll
    for (int d = 1; d < W; d <<= 1) to = max_f(to, __shfl_xor(to, d, W));
    if (to != -kInf) move(to);
    s = team_sum<W>(s);
    t = team_sum<W>(t);
  }
};

// a wave's list of the largest logits so far, larger first, equal ones by the
// lower class; entry j in lane j
struct Top {
  int key = kNone;
  int cls = 0;
  int size = 0;   // uniform
  float floor = -kInf;  // the last entry of a full list
  __device__ __forceinline__ void put(int k, int c, int top) {
    const int lane = threadIdx.x & 63;
    const int at = __popcll(__ballot(lane < size && (key > k || (key == k && cls < c))));
    const int up_k = __shfl_up(key, 1), up_c = __shfl_up(cls, 1);
    if (lane > at) {
      key = up_k;
      cls = up_c;
    } else if (lane == at) {
      key = k;
      cls = c;
    }
    size = size < top ? size + 1 : top;
    if (size == top) floor = value_of(__builtin_amdgcn_readlane(key, top - 1));
  }
  // N logits a lane, the class of lane l's j-th is base + l * N + j; those outside
  // [0, classes) are none.  Later calls have higher classes.
  template <int N>
  __device__ void take(const float (&x)[N], int base, int classes, int top) {
    int k[N];
    const int lane = threadIdx.x & 63;
    const int c0 = base + lane * N;
#pragma unroll
    for (int j = 0; j < N; ++j) k[j] = c0 + j >= 0 && c0 + j < classes ? key_of(x[j]) : kNone;
    for (;;) {
      int best = k[0];
#pragma unroll
      for (int j = 1; j < N; ++j) best = best > k[j] ? best : k[j];
      const int m = wave_max(best);
      if (m == kNone || (size == top && m <= __builtin_amdgcn_readlane(key, top - 1))) return;
      const int from = __ffsll((unsigned long long)__ballot(best == m)) - 1;
      int j0 = 0;
#pragma unroll
      for (int j = N - 1; j >= 0; --j) j0 = k[j] == m ? j : j0;
      const int c = __builtin_amdgcn_readlane(c0 + j0, from);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (lane == from && j == j0) k[j] = kNone;
      put(m, c, top);
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

__device__ __forceinline__ float log_of(float s) { return __logf(s); }

// log p of a logit from the row's statistics (R, log S); an empty row: -inf
__device__ __forceinline__ float logp_of(float x, float r, float ls) {
  return r == -kInf && ls == -kInf ? -kInf : (x - r) - ls;
}

template <typename T>
__device__ __forceinline__ void write_row(const RowOut& o, int64_t row, const T* x, int64_t classes,
                                          float r, float s, float t) {
  const float ls = s == 0.f ? -kInf : logf(s);
  o.stats[2 * row] = r;
  o.stats[2 * row + 1] = ls;
  o.entropy[row] = s == 0.f ? 0.f : ls - t / s;
  if (o.logp) {
    const int64_t c = o.target[row];
    o.logp[row] = c == o.ignore ? 0.f
                  : c >= 0 && c < classes ? logp_of(to_f32(x[c]), r, ls)
                                          : __builtin_nanf("");
  }
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
    if (l == 0) write_row(o, row, xr, classes, a.r, a.s, a.t);
    if (top) {
      const float ls = a.s == 0.f ? -kInf : logf(a.s);
      int k[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) k[j] = j * W + l < classes ? key_of(v[j]) : kNone;
      for (int n = 0; n < top; ++n) {
        int bk = kNone, bc = INT32_MAX;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (k[j] > bk) {
            bk = k[j];
            bc = j * W + l;
          }
        }
#pragma unroll
        for (int d = 1; d < W; d <<= 1) {
          const int ok = __shfl_xor(bk, d, W), oc = __shfl_xor(bc, d, W);
          if (ok > bk || (ok == bk && oc < bc)) {
            bk = ok;
            bc = oc;
          }
        }
        if (l == 0) {
          o.top_class[row * top + n] = bc;
          o.top_logp[row * top + n] = logp_of(value_of(bk), a.r, ls);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (bc == j * W + l) k[j] = kNone;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// more classes: W waves of a block a row, or a split of one
// ---------------------------------------------------------------------------
struct Partial {  // of a split, followed by its top list
  float r, s, t;
  int size;
};

// sums and top list of the elements [begin, end) of a row that this wave reads:
// wave w of W
template <typename T, int W>
__device__ __forceinline__ void scan_row(const T* xr, int begin, int end, int w, int top, Sums& a,
                                         Top& best) {
  constexpr int V = 16 / sizeof(T);
  constexpr int U = 4;
  const int lane = threadIdx.x & 63;
  float bound = -kInf;  // a vector whose largest logit is not above it needs no second look
  auto again = [&]() {
    bound = a.r + kSlack;
    if (top) bound = best.size == top ? (bound < best.floor ? bound : best.floor) : -kInf;
  };
  auto one = [&](const auto& x, int base) {  // base: the class of lane 0's first logit
    constexpr int N = sizeof(x) / sizeof(float);
    float m = x[0];
    if constexpr (N > 1) {
      m = max_f(x[0], x[1]);
#pragma unroll
      for (int j = 2; j + 1 < N; j += 2) m = max3_f(m, x[j], x[j + 1]);
    }
    if (__ballot(m > bound || (top && best.size < top))) {
      if (m > a.r + kSlack) a.move(m);
      if (top && __ballot(m > best.floor || best.size < top)) best.take(x, base, end, top);
      again();
    }
#pragma unroll
    for (int j = 0; j < N; ++j) a.add(x[j]);
  };
  // [begin, lo) and [hi, end): what the 16-byte vectors leave, one element a lane
  const int head = int((16 - (reinterpret_cast<uintptr_t>(xr + begin) & 15)) & 15) / int(sizeof(T));
  const int lo = begin + (head < end - begin ? head : end - begin);
  const int vecs = (end - lo) / V, hi = lo + vecs * V;
  if (w == 0 && lo > begin) {
    const float x[1] = {lane < lo - begin ? to_f32(xr[begin + lane]) : -kInf};
    one(x, lane < lo - begin ? begin : end);
  }
  const auto* p = reinterpret_cast<const Pack<T, V>*>(xr + lo);
  for (int v0 = w * 64; v0 < vecs; v0 += W * 64 * U) {
    Pack<T, V> q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + u * W * 64 + lane;
      if (v < vecs) q[u] = p[v];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = v0 + u * W * 64;
      if (v >= vecs) break;
      float x[V];
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] = v + lane < vecs ? to_f32(q[u].v[j]) : -kInf;
      // classes beyond hi belong to the tail: none here
      one(x, v + lane < vecs ? lo + v * V : end);
    }
  }
  if (w == 0 && hi < end) {
    const float x[1] = {lane < end - hi ? to_f32(xr[hi + lane]) : -kInf};
    one(x, hi);
  }
}

// the larger first, equal ones by the lower class: the top of ``n`` listed entries
template <typename F>
__device__ __forceinline__ void top_of_lists(const int2* list, int n, int top, F put) {
  const int lane = threadIdx.x & 63;
  int last_k = INT32_MAX, last_c = -1;
  for (int out = 0; out < top; ++out) {
    // the largest entry after the last one put
    int bk = kNone, bc = INT32_MAX;
    for (int i = lane; i < n; i += 64) {
      const int2 e = list[i];
      const bool after = e.x < last_k || (e.x == last_k && e.y > last_c);
      if (after && (e.x > bk || (e.x == bk && e.y < bc))) {
        bk = e.x;
        bc = e.y;
      }
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int ok = __shfl_xor(bk, d), oc = __shfl_xor(bc, d);
      if (ok > bk || (ok == bk && oc < bc)) {
        bk = ok;
        bc = oc;
      }
    }
    last_k = bk;
    last_c = bc;
    put(out, bk, bc);
  }
}

template <typename T, int W, bool SPLIT>
__global__ void __launch_bounds__(kThreads) k_fwd_wide(const T* __restrict__ x, int64_t rows,
                                                       int classes, int64_t stride, int top,
                                                       int splits, int per_split,
                                                       Partial* __restrict__ part,
                                                       int2* __restrict__ part_top, RowOut o) {
  __shared__ Partial sums[kWaves];
  __shared__ int2 lists[W > 1 ? W * kMaxTop : 1];
  const int lane = threadIdx.x & 63, wave = wave_uniform(threadIdx.x >> 6);
  const int64_t jobs = rows * (SPLIT ? splits : 1);
  const int64_t step = int64_t(gridDim.x) * (kWaves / W);
  // every wave of a block runs the same number of iterations (a barrier inside)
  for (int64_t job0 = int64_t(blockIdx.x) * (kWaves / W); job0 < jobs; job0 += step) {
    const int64_t job = job0 + (W > 1 ? 0 : wave);
    if (W == 1 && job >= jobs) break;
    const int64_t row = SPLIT ? job / splits : job;
    const int begin = SPLIT ? int(job - row * splits) * per_split : 0;
    const int end = SPLIT ? (begin + per_split < classes ? begin + per_split : classes) : classes;
    const T* xr = x + row * stride;
    Sums a;
    Top best;
    scan_row<T, W>(xr, begin, end, W > 1 ? wave : 0, top, a, best);
    a.join<64>();
    if (W > 1) {
      if (lane == 0) sums[wave] = {a.r, a.s, a.t, best.size};
      if (lane < top) lists[wave * top + lane] = {lane < best.size ? best.key : kNone, best.cls};
      __syncthreads();
      if (wave == 0) {
        a = Sums();
        if (lane < W) {
          a.r = sums[lane].r;
          a.s = sums[lane].s;
          a.t = sums[lane].t;
        }
        a.join<W>();
      }
    }
    if (W == 1 || wave == 0) {
      if (SPLIT) {
        if (lane == 0) part[job] = {a.r, a.s, a.t, 0};
      } else if (lane == 0) {
        write_row(o, row, xr, classes, a.r, a.s, a.t);
      }
      if (top) {
        const float r = __shfl(a.r, 0), s = __shfl(a.s, 0);
        const float ls = s == 0.f ? -kInf : logf(s);
        auto put = [&](int j, int k, int c) {
          if (lane == 0) {
            if (SPLIT) {
              part_top[job * top + j] = {k, c};
            } else {
              o.top_class[row * top + j] = c;
              o.top_logp[row * top + j] = logp_of(value_of(k), r, ls);
            }
          }
        };
        if (W > 1) {
          top_of_lists(lists, W * top, top, put);
        } else if (lane < top) {
          o.top_class[row * top + lane] = best.cls;
          o.top_logp[row * top + lane] = logp_of(value_of(best.key), r, ls);
        }
      }
    }
    if (W > 1) __syncthreads();  // the next row writes the lists
  }
}

// a wave a row: the splits' sums and lists
template <typename T>
__global__ void __launch_bounds__(kWave) k_fwd_join(const T* __restrict__ x, int64_t rows,
                                                    int classes, int64_t stride, int top,
                                                    int splits, const Partial* __restrict__ part,
                                                    const int2* __restrict__ part_top, RowOut o) {
  const int lane = threadIdx.x;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    Sums a;
    for (int i = lane; i < splits; i += 64) {
      const Partial p = part[row * splits + i];
      if (p.r > a.r) a.move(p.r);
      Sums b;
      b.r = p.r;
      b.s = p.s;
      b.t = p.t;
      if (p.r != -kInf) b.move(a.r);
      a.s += b.s;
      a.t += b.t;
    }
    a.join<64>();
    if (lane == 0) write_row(o, row, x + row * stride, classes, a.r, a.s, a.t);
    const float ls = a.s == 0.f ? -kInf : logf(a.s);
    if (top)
      top_of_lists(part_top + row * splits * top, splits * top, top, [&](int j, int k, int c) {
        if (lane == 0) {
          o.top_class[row * top + j] = c;
          o.top_logp[row * top + j] = logp_of(value_of(k), a.r, ls);
        }
      });
  }
}

// how many blocks share a row, and the classes of one (a multiple of 16)
inline int splits_of(int64_t rows, int64_t classes) {
  if (classes <= kWaveRow || rows >= kFill) return 1;
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

template <typename T, int V, bool NARROW>
__global__ void __launch_bounds__(kThreads) k_bwd(const T* __restrict__ x, int64_t rows,
                                                  int classes, int64_t stride, int parts,
                                                  int per_part, BwdArgs b, T* __restrict__ out) {
  if (NARROW) {
    // one logit a thread, in the output's order
    const int64_t n = rows * classes;
    for (int64_t e = int64_t(blockIdx.x) * kThreads + threadIdx.x; e < n;
         e += int64_t(gridDim.x) * kThreads) {
      const int64_t row = e / classes;
      const int c = int(e - row * classes);
      const BwdRow w = bwd_row(b, row, classes);
      float g = w.empty ? 0.f : bwd_dense(w, to_f32(x[row * stride + c]));
      if (!w.empty && c == w.target) g += w.given;
      if (b.g_top && !w.empty)
        for (int j = 0; j < b.top; ++j)
          if (b.top_class[row * b.top + j] == c) g += b.g_top[row * b.top + j];
      out[e] = from_f32<T>(g);
    }
    return;
  }
  for (int64_t job = blockIdx.x; job < rows * parts; job += gridDim.x) {
    const int64_t row = job / parts;
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
      for (int v = threadIdx.x; v < vecs; v += kThreads) {
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
    for (int c = begin + threadIdx.x; c < lo; c += kThreads) at(c);
    for (int c = lo + vecs * V + threadIdx.x; c < end; c += kThreads) at(c);
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
  const int s = splits_of(rows, classes);
  if (s == 1) return 0;
  Sizer z;
  z.take<Partial>(size_t(rows) * s);
  z.take<int2>(size_t(rows) * s * top);
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
  const int splits = splits_of(rows, classes);
  Partial* part = nullptr;
  int2* part_top = nullptr;
  if (splits > 1) {
    Carve c(ws, ws_bytes);
    part = c.take<Partial>(size_t(rows) * splits);
    part_top = c.take<int2>(size_t(rows) * splits * top);
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
    } else if (n <= kWaveRow) {
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
    if (n < 512) {
      const int64_t blocks = (rows * n + kThreads - 1) / kThreads;
      k_bwd<T, 1, true><<<int(blocks < 65536 ? blocks : 65536), kThreads, 0, stream>>>(
          x, rows, n, row_stride, 1, n, b, g);
    } else {
      const int parts = (n + 8191) / 8192, per = int(align_up(size_t((n + parts - 1) / parts), 16));
      const int64_t jobs = rows * parts;
      const int grid = int(jobs < 65536 ? jobs : 65536);
      // 16-byte vectors where every row of both starts at the same place of one
      const bool same = (reinterpret_cast<uintptr_t>(x) - reinterpret_cast<uintptr_t>(g)) % 16 == 0 &&
                        (rows == 1 || (row_stride - classes) * int64_t(sizeof(T)) % 16 == 0);
      if (same)
        k_bwd<T, V, false><<<grid, kThreads, 0, stream>>>(x, rows, n, row_stride, parts, per, b, g);
      else
        k_bwd<T, 1, false><<<grid, kThreads, 0, stream>>>(x, rows, n, row_stride, parts, per, b, g);
    }
    GFD_LAUNCH_CHECK();
    return GFD_OK;
  });
}

}  // extern "C"
