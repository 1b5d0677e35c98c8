// gfd_group_norm.hip -- group norm with an activation over node rows (channels
// last), forward and backward, dense or ragged segments of rows.
//
//   xhat = (x - mean_sg) rstd_sg,  z = xhat w + b,  y = act(z)
//   dz = dy act'(z),  A = mean_sg(w dz),  B = mean_sg(w dz xhat)
//   dx = rstd (w dz - A - xhat B),  dw = sum dz xhat,  db = sum dz
//
// Bound by memory: x in and y out (backward: x and dy in, dx out), with a few
// dozen operations an element.  A thread holds one vector of V channels of a
// row, V dividing the channels of a group, so that a vector lies in one group;
// sums are fp64 throughout (x and x^2: a large mean costs nothing).
//   * A short segment is normalised by one team of threads (k_team): its rows
//     are read twice, the second time from cache, in one launch.
//   * A long one is cut into tiles of rows: k_sums writes each tile's column
//     sums, k_stats joins those of a segment and group in a fixed order, k_apply
//     writes the result.  A ragged segment is long when it has more rows than a
//     tile; then it holds the first or the last row of every tile that it
//     touches, so that a tile meets at most two of them and finds them by two
//     binary searches, however many segments there are.
//   * The weight and bias gradients are the column sums of all blocks and tiles,
//     added in a fixed order by k_columns.
#include "gfd_rowops.h"

using namespace gfd;

namespace {

constexpr int kMaxChannels = 2048;
constexpr int kTeamBlocks = 1024;
constexpr int kMaxTeam = 1024;  // threads

struct Norm {
  const void* x;
  const void* dy;
  void* out;  // y or dx
  const int64_t* ptr;
  int64_t segments, length, row_stride, seg_stride;
  const void* w;
  const void* b;
  double* stats;   // [segments, groups, 2]
  double2* part;   // column sums
  double2* mom;    // backward: A, B of a segment and group
  double eps;
  int channels, groups, w_f32, act;
  int tile;        // rows of a tile; ragged segments up to it are short
  int tiles;       // of one segment (dense) or of all rows (ragged)
  int part0;       // first row of ``part`` that the teams write (backward)
  int cols, rows;  // team: threads over a row's vectors, over rows
  int zero_rest;   // ragged: k_apply clears the rows of no segment
};

// ---------------------------------------------------------------------------
// segments and tiles
// ---------------------------------------------------------------------------
__device__ __forceinline__ int64_t ptr_at(const Norm& n, int64_t s) {
  const int64_t v = n.ptr[s];
  return v < 0 ? 0 : v > n.length ? n.length : v;
}

// the rows of segment s in the layout's numbering
__device__ __forceinline__ void segment_rows(const Norm& n, int64_t s, int64_t& r0, int64_t& r1) {
  if (n.ptr) {
    r0 = ptr_at(n, s);
    r1 = ptr_at(n, s + 1);
  } else {
    r0 = s * n.length;
    r1 = r0 + n.length;
  }
}

// the last segment that starts at or before row r, -1: none
__device__ __forceinline__ int64_t segment_of(const Norm& n, int64_t r) {
  int64_t lo = -1, hi = n.segments;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (ptr_at(n, mid) <= r) lo = mid;
    else hi = mid;
  }
  return lo;
}

struct Piece {
  int64_t seg, r0, r1;  // rows [r0, r1) of segment seg
};

// the pieces of long segments in a tile; piece i's sums go to row 2 t + i (ragged) or t of ``part``
__device__ __forceinline__ int pieces_of(const Norm& n, int64_t t, Piece (&p)[2]) {
  if (!n.ptr) {
    const int64_t s = t / n.tiles, r0 = s * n.length, k = (t - s * n.tiles) * n.tile;
    const int64_t k1 = k + n.tile < n.length ? k + n.tile : n.length;
    p[0] = {s, r0 + k, r0 + k1};
    return 1;
  }
  const int64_t a = t * n.tile, e = a + n.tile < n.length ? a + n.tile : n.length;
  const int64_t s0 = segment_of(n, a), s1 = segment_of(n, e - 1);
  int found = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t s = i == 0 ? s0 : s1;
    p[i] = {-1, 0, 0};
    if (s < 0 || (i == 1 && s1 == s0)) continue;
    int64_t r0, r1;
    segment_rows(n, s, r0, r1);
    if (r1 - r0 <= n.tile) continue;
    r0 = r0 < a ? a : r0;
    r1 = r1 > e ? e : r1;
    if (r0 < r1) {
      p[i] = {s, r0, r1};
      found = i + 1;
    }
  }
  return found;
}

template <typename T>
__device__ __forceinline__ const T* row_in(const Norm& n, const void* base, int64_t seg, int64_t r) {
  const T* p = static_cast<const T*>(base);
  return n.ptr ? p + r * n.row_stride
               : p + seg * n.seg_stride + (r - seg * n.length) * n.row_stride;
}

// ---------------------------------------------------------------------------
// element arithmetic
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float affine_at(const void* p, int f32, int c, float none) {
  if (!p) return none;
  return f32 ? static_cast<const float*>(p)[c] : to_f32(static_cast<const T*>(p)[c]);
}

// activation and, where D is not null, its derivative at z
__device__ __forceinline__ float activate(float z, int act, float* d) {
  switch (act) {
    case GFD_ACT_RELU:
      if (d) *d = z > 0.f ? 1.f : 0.f;
      return z > 0.f ? z : z != z ? z : 0.f;
    case GFD_ACT_SILU: {
      const float p = 1.f / (1.f + __expf(-z));
      if (d) *d = p * (1.f + z * (1.f - p));
      return z * p;
    }
    case GFD_ACT_GELU: {
      const float p = 0.5f * (1.f + erff(z * 0.70710678118654752f));
      if (d) *d = p + z * __expf(-0.5f * z * z) * 0.39894228040143268f;
      return z * p;
    }
    default:
      if (d) *d = 1.f;
      return z;
  }
}

struct Moments {
  double mean, rstd;
  float hi, lo, r;  // mean = hi + lo
  __device__ __forceinline__ Moments(double m, double s) : mean(m), rstd(s) {
    hi = float(m);
    lo = float(m - double(hi));
    r = float(s);
  }
  __device__ __forceinline__ float xhat(float x) const { return ((x - hi) - lo) * r; }
  // xhat w + b; where it is too near 0 for fp32 to tell relu's side, from fp64
  __device__ __forceinline__ float z(float x, float xh, float w, float b, int act) const {
    const float p = xh * w, v = p + b;
    if (act == GFD_ACT_RELU && fabsf(v) <= 1e-5f * (fabsf(p) + fabsf(b)))
      return float((double(x) - mean) * rstd * double(w) + double(b));
    return v;
  }
};

template <typename T, int V>
struct Affine {
  float w[V], b[V];
  __device__ __forceinline__ void load(const Norm& n, int col) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      w[j] = affine_at<T>(n.w, n.w_f32, col * V + j, 1.f);
      b[j] = affine_at<T>(n.b, n.w_f32, col * V + j, 0.f);
    }
  }
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> forward(const Pack<T, V>& x, const Moments& m,
                                              const Affine<T, V>& a, int act) {
  Pack<T, V> y;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float v = to_f32(x.v[j]), xh = m.xhat(v);
    y.v[j] = from_f32<T>(activate(m.z(v, xh, a.w[j], a.b[j], act), act, nullptr));
  }
  return y;
}

// dz and xhat of one vector
template <typename T, int V>
__device__ __forceinline__ void slope(const Pack<T, V>& x, const Pack<T, V>& dy, const Moments& m,
                                      const Affine<T, V>& a, int act, float (&dz)[V],
                                      float (&xh)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float v = to_f32(x.v[j]);
    xh[j] = m.xhat(v);
    float d;
    activate(m.z(v, xh[j], a.w[j], a.b[j], act), act, &d);
    dz[j] = to_f32(dy.v[j]) * d;
  }
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> backward(const float (&dz)[V], const float (&xh)[V],
                                               const Moments& m, const Affine<T, V>& a, float ma,
                                               float mb) {
  Pack<T, V> g;
#pragma unroll
  for (int j = 0; j < V; ++j) g.v[j] = from_f32<T>(m.r * (a.w[j] * dz[j] - ma - xh[j] * mb));
  return g;
}

// mean and 1 / sqrt(var + eps) from the sums of x and x^2 over n elements
__device__ __forceinline__ double2 moments_of(double s, double q, double n, double eps) {
  const double mean = s / n;
  double var = q / n - mean * mean;
  if (var < 0.0) var = 0.0;
  return {mean, 1.0 / sqrt(var + eps)};
}

// ---------------------------------------------------------------------------
// short segments: a team of cols x rows threads each
// ---------------------------------------------------------------------------
template <typename T, int V, int NC, bool BWD>
__global__ void __launch_bounds__(kMaxTeam) k_team(const Norm n) {
  extern __shared__ double2 lds[];
  double2* red = lds;                 // [blockDim]
  double2* col_sum = lds + blockDim.x;  // [teams][vecs]
  using P = Pack<T, V>;
  const int vecs = n.channels / V, gv = vecs / n.groups;
  const int size = n.cols * n.rows, teams = blockDim.x / size;
  const int c = threadIdx.x % n.cols, tr = threadIdx.x / n.cols % n.rows, team = threadIdx.x / size;
  Affine<T, V> aff[NC];
  double dw[NC][V] = {}, db[NC][V] = {};
#pragma unroll
  for (int k = 0; k < NC; ++k)
    if (c + k * n.cols < vecs) aff[k].load(n, c + k * n.cols);
  for (int64_t s0 = int64_t(blockIdx.x) * teams; s0 < n.segments; s0 += int64_t(gridDim.x) * teams) {
    const int64_t seg = s0 + team;
    int64_t r0 = 0, r1 = 0;
    if (seg < n.segments) {
      segment_rows(n, seg, r0, r1);
      if (n.ptr && r1 - r0 > n.tile) r1 = r0;  // a long one: not here
    }
    // sums of each column: x and x^2, or w dz and w dz xhat
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int col = c + k * n.cols;
      double a = 0.0, b = 0.0;
      if (col < vecs && r0 < r1) {
        double mean = 0.0, rstd = 0.0;
        if (BWD) {
          const double* st = n.stats + 2 * (seg * n.groups + col / gv);
          mean = st[0];
          rstd = st[1];
        }
        const Moments m(mean, rstd);
        for (int64_t r = r0 + tr; r < r1; r += n.rows) {
          const P x = *reinterpret_cast<const P*>(row_in<T>(n, n.x, seg, r) + col * V);
          if (BWD) {
            const P dy = *reinterpret_cast<const P*>(static_cast<const T*>(n.dy) + r * n.channels + col * V);
            float dz[V], xh[V];
            slope<T, V>(x, dy, m, aff[k], n.act, dz, xh);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const double e = double(dz[j]), f = e * double(xh[j]);
              db[k][j] += e;
              dw[k][j] += f;
              a += double(aff[k].w[j]) * e;
              b += double(aff[k].w[j]) * f;
            }
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const double v = double(to_f32(x.v[j]));
              a += v;
              b += v * v;
            }
          }
        }
      }
      if (n.rows > 1) {
        red[threadIdx.x] = {a, b};
        __syncthreads();
        if (tr == 0)
          for (int i = 1; i < n.rows; ++i) {
            a += red[threadIdx.x + i * n.cols].x;
            b += red[threadIdx.x + i * n.cols].y;
          }
      }
      if (tr == 0 && col < vecs) col_sum[team * vecs + col] = {a, b};
      __syncthreads();
    }
    // of each group, in place of its first column
    for (int i = threadIdx.x; i < teams * n.groups; i += blockDim.x) {
      const int tm = i / n.groups, g = i - tm * n.groups;
      const int64_t sg = s0 + tm;
      int64_t q0 = 0, q1 = 0;
      if (sg < n.segments) {
        segment_rows(n, sg, q0, q1);
        if (n.ptr && q1 - q0 > n.tile) q1 = q0;
      }
      if (q0 >= q1) continue;
      double2* cs = col_sum + tm * vecs + g * gv;
      double a = 0.0, b = 0.0;
      for (int k = 0; k < gv; ++k) {
        a += cs[k].x;
        b += cs[k].y;
      }
      const double count = double(q1 - q0) * (n.channels / n.groups);
      if (BWD) {
        cs[0] = {a / count, b / count};
      } else {
        const double2 m = moments_of(a, b, count, n.eps);
        cs[0] = m;
        if (n.stats) {
          n.stats[2 * (sg * n.groups + g)] = m.x;
          n.stats[2 * (sg * n.groups + g) + 1] = m.y;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int col = c + k * n.cols;
      if (col < vecs && r0 < r1) {
        const double2 v = col_sum[team * vecs + col / gv * gv];
        double mean = v.x, rstd = v.y;
        if (BWD) {
          const double* st = n.stats + 2 * (seg * n.groups + col / gv);
          mean = st[0];
          rstd = st[1];
        }
        const Moments m(mean, rstd);
        for (int64_t r = r0 + tr; r < r1; r += n.rows) {
          const P x = *reinterpret_cast<const P*>(row_in<T>(n, n.x, seg, r) + col * V);
          P* out = reinterpret_cast<P*>(static_cast<T*>(n.out) + r * n.channels + col * V);
          if (BWD) {
            const P dy = *reinterpret_cast<const P*>(static_cast<const T*>(n.dy) + r * n.channels + col * V);
            float dz[V], xh[V];
            slope<T, V>(x, dy, m, aff[k], n.act, dz, xh);
            *out = backward<T, V>(dz, xh, m, aff[k], float(v.x), float(v.y));
          } else {
            *out = forward<T, V>(x, m, aff[k], n.act);
          }
        }
      }
    }
    __syncthreads();
  }
  if (BWD) {  // this block's column sums of dz and dz xhat
    double2* part = n.part + int64_t(n.part0 + blockIdx.x) * n.channels;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int col = c + k * n.cols;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        red[threadIdx.x] = {db[k][j], dw[k][j]};
        __syncthreads();
        if (threadIdx.x < n.cols && col < vecs) {
          double2 t = red[threadIdx.x];
          for (int i = threadIdx.x + n.cols; i < int(blockDim.x); i += n.cols) {
            t.x += red[i].x;
            t.y += red[i].y;
          }
          part[col * V + j] = t;
        }
        __syncthreads();
      }
    }
  }
}

// ---------------------------------------------------------------------------
// long segments
// ---------------------------------------------------------------------------
constexpr int kTileThreads = 256;

// column sums of a tile: forward [slot][vecs] of x and x^2, backward [slot][channels] of dz and
// dz xhat; ragged tiles have two slots, an unused one is 0
template <typename T, int V, bool BWD>
__global__ void __launch_bounds__(kTileThreads) k_sums(const Norm n) {
  using P = Pack<T, V>;
  constexpr int S = BWD ? V : 1;
  __shared__ double2 red[kTileThreads];
  const int vecs = n.channels / V, gv = vecs / n.groups;
  const int c = threadIdx.x % n.cols, tr = threadIdx.x / n.cols, rows = kTileThreads / n.cols;
  const int col = blockIdx.y * n.cols + c;
  const int64_t t = blockIdx.x;
  Affine<T, V> aff;
  if (BWD && col < vecs) aff.load(n, col);
  Piece p[2];
  const int found = pieces_of(n, t, p);
  for (int i = 0; i < (n.ptr ? 2 : 1); ++i) {
    double a[S] = {}, b[S] = {};
    if (i < found && p[i].seg >= 0 && col < vecs) {
      double mean = 0.0, rstd = 0.0;
      if (BWD) {
        const double* st = n.stats + 2 * (p[i].seg * n.groups + col / gv);
        mean = st[0];
        rstd = st[1];
      }
      const Moments m(mean, rstd);
#pragma unroll 4
      for (int64_t r = p[i].r0 + tr; r < p[i].r1; r += rows) {
        const P x = *reinterpret_cast<const P*>(row_in<T>(n, n.x, p[i].seg, r) + col * V);
        if (BWD) {
          const P dy = *reinterpret_cast<const P*>(static_cast<const T*>(n.dy) + r * n.channels + col * V);
          float dz[V], xh[V];
          slope<T, V>(x, dy, m, aff, n.act, dz, xh);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            a[j % S] += double(dz[j]);
            b[j % S] += double(dz[j]) * double(xh[j]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const double v = double(to_f32(x.v[j]));
            a[0] += v;
            b[0] += v * v;
          }
        }
      }
    }
    const int64_t slot = n.ptr ? 2 * t + i : t;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      red[threadIdx.x] = {a[j], b[j]};
      __syncthreads();
      if (tr == 0 && col < vecs) {
        double2 v = red[c];
        for (int k = 1; k < rows; ++k) {
          v.x += red[c + k * n.cols].x;
          v.y += red[c + k * n.cols].y;
        }
        n.part[slot * (BWD ? n.channels : vecs) + col * S + j] = v;
      }
      __syncthreads();
    }
  }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// a wave for each long segment and group: its tiles' sums
template <typename T, int V, bool BWD>
__global__ void __launch_bounds__(kWave) k_stats(const Norm n) {
  const int vecs = n.channels / V, per = n.channels / n.groups;
  const int width = BWD ? n.channels : vecs, each = BWD ? per : vecs / n.groups;
  for (int64_t job = blockIdx.x; job < n.segments * n.groups; job += gridDim.x) {
    const int64_t s = job / n.groups;
    const int g = int(job - s * n.groups);
    int64_t r0, r1, first, count;
    segment_rows(n, s, r0, r1);
    if (n.ptr) {
      if (r1 - r0 <= n.tile) continue;
      first = r0 / n.tile;
      count = (r1 - 1) / n.tile - first + 1;
    } else {
      first = s * n.tiles;
      count = n.tiles;
    }
    double a = 0.0, b = 0.0;
    for (int64_t i = threadIdx.x; i < count * each; i += kWave) {
      const int64_t k = i / each;
      const int c = int(i - k * each) + g * each;
      int64_t slot = first + k;
      // ragged: the second slot where the segment starts inside the tile
      if (n.ptr) slot = 2 * slot + (r0 > slot * n.tile ? 1 : 0);
      const double2 v = n.part[slot * width + c];
      const double w = BWD ? double(affine_at<T>(n.w, n.w_f32, c, 1.f)) : 1.0;
      a += w * v.x;
      b += w * v.y;
    }
    a = wave_sum(a);
    b = wave_sum(b);
    if (threadIdx.x == 0) {
      const double total = double(r1 - r0) * per;
      if (BWD) {
        n.mom[job] = {a / total, b / total};
      } else {
        const double2 m = moments_of(a, b, total, n.eps);
        n.stats[2 * job] = m.x;
        n.stats[2 * job + 1] = m.y;
      }
    }
  }
}

template <typename T, int V, bool BWD>
__global__ void __launch_bounds__(kTileThreads) k_apply(const Norm n) {
  using P = Pack<T, V>;
  const int vecs = n.channels / V, gv = vecs / n.groups;
  const int c = threadIdx.x % n.cols, tr = threadIdx.x / n.cols, rows = kTileThreads / n.cols;
  const int col = blockIdx.y * n.cols + c;
  if (col >= vecs) return;
  const int64_t t = blockIdx.x;
  Affine<T, V> aff;
  aff.load(n, col);
  Piece p[2];
  const int found = pieces_of(n, t, p);
  for (int i = 0; i < found; ++i) {
    if (p[i].seg < 0) continue;
    const int64_t job = p[i].seg * n.groups + col / gv;
    const Moments m(n.stats[2 * job], n.stats[2 * job + 1]);
    float ma = 0.f, mb = 0.f;
    if (BWD) {
      ma = float(n.mom[job].x);
      mb = float(n.mom[job].y);
    }
#pragma unroll 4
    for (int64_t r = p[i].r0 + tr; r < p[i].r1; r += rows) {
      const P x = *reinterpret_cast<const P*>(row_in<T>(n, n.x, p[i].seg, r) + col * V);
      P* out = reinterpret_cast<P*>(static_cast<T*>(n.out) + r * n.channels + col * V);
      if (BWD) {
        const P dy = *reinterpret_cast<const P*>(static_cast<const T*>(n.dy) + r * n.channels + col * V);
        float dz[V], xh[V];
        slope<T, V>(x, dy, m, aff, n.act, dz, xh);
        *out = backward<T, V>(dz, xh, m, aff, ma, mb);
      } else {
        *out = forward<T, V>(x, m, aff, n.act);
      }
    }
  }
  if (n.ptr) {  // the rows of no segment
    const int64_t a = t * n.tile, e = a + n.tile < n.length ? a + n.tile : n.length;
    const int64_t first = ptr_at(n, 0), last = ptr_at(n, n.segments);
    for (int64_t r = a + tr; r < e; r += rows)
      if (r < first || r >= last)
        *reinterpret_cast<P*>(static_cast<T*>(n.out) + r * n.channels + col * V) = P{};
  }
}

// the weight and bias gradients: a channel's column sums of all slots in a fixed order
template <typename T>
__global__ void __launch_bounds__(256) k_columns(const double2* __restrict__ part, int64_t slots,
                                                 int channels, int w_f32, void* dw, void* db) {
  __shared__ double2 red[256];
  const int c = blockIdx.x * 8 + (threadIdx.x & 7), k = threadIdx.x >> 3;
  double2 s = {0.0, 0.0};
  if (c < channels)
    for (int64_t i = k; i < slots; i += 32) {
      const double2 v = part[i * channels + c];
      s.x += v.x;
      s.y += v.y;
    }
  red[threadIdx.x] = s;
  __syncthreads();
  if (k == 0 && c < channels) {
    for (int i = 1; i < 32; ++i) {
      s.x += red[threadIdx.x + 8 * i].x;
      s.y += red[threadIdx.x + 8 * i].y;
    }
    if (db) {
      if (w_f32) static_cast<float*>(db)[c] = float(s.x);
      else static_cast<T*>(db)[c] = from_f32<T>(float(s.x));
    }
    if (dw) {
      if (w_f32) static_cast<float*>(dw)[c] = float(s.y);
      else static_cast<T*>(dw)[c] = from_f32<T>(float(s.y));
    }
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
inline int pow2_up(int64_t v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

// how a call is cut; depends on shapes alone, so that the workspace query agrees with the call
struct Cut {
  bool team, tiled;
  int tile;
  int64_t tiles;   // of a segment (dense) or of all rows (ragged)
  int64_t slots;   // tile slots
  int64_t teams;   // upper bound of the team kernel's blocks
};

Cut cut_of(int64_t segments, int64_t length, bool ragged) {
  Cut c;
  const int64_t rows = ragged ? length : segments * length;
  // tiles: about 2048 of them, 32 to 512 rows
  int64_t tile = pow2_up((rows + 2047) / 2048);
  tile = tile < 32 ? 32 : tile > 512 ? 512 : tile;
  c.tile = int(tile);
  if (ragged) {
    c.team = c.tiled = true;
    c.tiles = (length + tile - 1) / tile;
    c.slots = 2 * c.tiles;
  } else {
    c.team = length <= 32 || segments >= kTeamBlocks;
    c.tiled = !c.team;
    c.tiles = (length + tile - 1) / tile;
    c.slots = c.tiled ? segments * c.tiles : 0;
  }
  c.teams = c.team ? (segments < kTeamBlocks ? segments : kTeamBlocks) : 0;
  return c;
}

bool shape_ok(int64_t segments, int64_t length, int channels, int groups) {
  return segments >= 0 && length >= 0 && channels >= 1 && groups >= 1 && channels % groups == 0 &&
         segments <= (int64_t(1) << 40) && length <= (int64_t(1) << 40);
}

// the widest vector that divides a group's channels and that every row starts at
int vector_of(int64_t per_group, size_t size, const void* const* ptrs, int n, int64_t row_stride,
              int64_t seg_stride) {
  int v = int(16 / size);
  for (; v > 1; v >>= 1) {
    bool ok = per_group % v == 0 && row_stride % v == 0 && seg_stride % v == 0;
    for (int i = 0; i < n; ++i) ok = ok && aligned_to(ptrs[i], size * v);
    if (ok) break;
  }
  return v;
}

template <typename F>
gfd_status with_vector(int v, F f) {
  switch (v) {
    case 8: return f(std::integral_constant<int, 8>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 2: return f(std::integral_constant<int, 2>{});
    default: return f(std::integral_constant<int, 1>{});
  }
}

template <typename T, int V, bool BWD>
gfd_status launch(Norm n, const Cut& c, int64_t* team_blocks, hipStream_t stream) {
  const int vecs = n.channels / V;
  *team_blocks = 0;
  if (c.team && n.segments > 0) {
    const int nc = vecs > kMaxTeam ? 2 : 1;
    n.cols = pow2_up((vecs + nc - 1) / nc);
    const int block = n.cols > 256 ? n.cols : 256;
    // threads over the rows: as many as a segment has, of the mean length when ragged
    const int64_t mean = n.ptr ? (n.length + n.segments - 1) / n.segments : n.length;
    const int most = block / n.cols, want = pow2_up(mean < most ? (mean < 1 ? 1 : mean) : most);
    n.rows = want < most ? want : most;
    const int teams = block / (n.cols * n.rows);
    int64_t grid = (n.segments + teams - 1) / teams;
    grid = grid < c.teams ? grid : c.teams;
    *team_blocks = grid;
    const size_t lds = sizeof(double2) * (size_t(block) + size_t(teams) * vecs);
    if (nc == 1)
      k_team<T, V, 1, BWD><<<int(grid), block, lds, stream>>>(n);
    else if constexpr (V == 1)  // more vectors than threads
      k_team<T, V, 2, BWD><<<int(grid), block, lds, stream>>>(n);
    GFD_LAUNCH_CHECK();
  }
  if (c.tiled && c.slots > 0) {
    n.cols = pow2_up(vecs < kTileThreads ? vecs : kTileThreads);
    const int64_t tiles = n.ptr ? c.tiles : n.segments * c.tiles;
    const dim3 grid(unsigned(tiles), unsigned((vecs + n.cols - 1) / n.cols));
    k_sums<T, V, BWD><<<grid, kTileThreads, 0, stream>>>(n);
    GFD_LAUNCH_CHECK();
    const int64_t jobs = n.segments * n.groups;
    if (jobs > 0) k_stats<T, V, BWD><<<int(jobs < 65536 ? jobs : 65536), kWave, 0, stream>>>(n);
    GFD_LAUNCH_CHECK();
    k_apply<T, V, BWD><<<grid, kTileThreads, 0, stream>>>(n);
    GFD_LAUNCH_CHECK();
  }
  return GFD_OK;
}

gfd_status check(const void* x, int dtype, int64_t segments, int64_t length, int channels,
                 int groups, int64_t row_stride, int64_t seg_stride, const void* weight,
                 const void* bias, int w_dtype, int act) {
  if (!float_dtype(dtype) || !shape_ok(segments, length, channels, groups)) return GFD_ERR_ARGUMENT;
  if (channels > kMaxChannels) return GFD_ERR_UNSUPPORTED;
  if (w_dtype != dtype && w_dtype != GFD_DTYPE_F32) return GFD_ERR_ARGUMENT;
  if (act < GFD_ACT_NONE || act > GFD_ACT_GELU || row_stride < 0 || seg_stride < 0)
    return GFD_ERR_ARGUMENT;
  if (!aligned_to(x, dtype_size(dtype)) || !aligned_to(weight, dtype_size(w_dtype)) ||
      !aligned_to(bias, dtype_size(w_dtype)))
    return GFD_ERR_ARGUMENT;
  return GFD_OK;
}

// tiles and slots are counted in 32 bits by the grid
bool grid_ok(const Cut& c, int64_t segments, bool ragged) {
  const int64_t tiles = ragged ? c.tiles : c.tiled ? segments * c.tiles : 0;
  return tiles < (int64_t(1) << 31);
}

}  // namespace

extern "C" {

size_t gfd_group_norm_workspace_size(int64_t segments, int64_t length, int ragged, int channels,
                                     int groups, int backward) {
  if (!shape_ok(segments, length, channels, groups) || channels > kMaxChannels) return 0;
  if (!ragged && (segments == 0 || length == 0)) return 0;
  const Cut c = cut_of(segments, length, ragged != 0);
  Sizer z;
  z.take<double2>(size_t(c.slots + (backward ? c.teams : 0)) * channels);
  z.take<double2>(c.tiled ? size_t(segments) * groups : 0);
  return z.off;
}

gfd_status gfd_group_norm_fwd(const void* x, int dtype, int64_t segments, int64_t length,
                              const int64_t* ptr, int channels, int groups, int64_t row_stride,
                              int64_t seg_stride, const void* weight, const void* bias,
                              int w_dtype, double eps, int act, void* y, double* stats, void* ws,
                              size_t ws_bytes, gfd_stream_t stream) {
  gfd_status st = check(x, dtype, segments, length, channels, groups, row_stride, seg_stride,
                        weight, bias, w_dtype, act);
  if (st != GFD_OK) return st;
  if (!(eps >= 0.0)) return GFD_ERR_ARGUMENT;
  if (length == 0 || (!ptr && segments == 0)) return GFD_OK;
  if (!x || !y || !aligned_to(y, dtype_size(dtype))) return GFD_ERR_ARGUMENT;
  const Cut c = cut_of(segments, length, ptr != nullptr);
  if (!grid_ok(c, segments, ptr != nullptr)) return GFD_ERR_UNSUPPORTED;
  Carve cv(ws, ws_bytes);
  Norm n = {};
  if (c.slots > 0 || c.tiled) {
    n.part = cv.take<double2>(size_t(c.slots) * channels);
    n.mom = cv.take<double2>(c.tiled ? size_t(segments) * groups : 0);
    if (!cv.ok) return GFD_ERR_WORKSPACE;
  }
  n.x = x;
  n.out = y;
  n.ptr = ptr;
  n.segments = segments;
  n.length = length;
  n.row_stride = row_stride;
  n.seg_stride = seg_stride;
  n.w = weight;
  n.b = bias;
  // the tile kernels hand the statistics on: without a place of the caller's, through ``mom``
  n.stats = stats ? stats : c.tiled ? reinterpret_cast<double*>(n.mom) : nullptr;
  n.eps = eps;
  n.channels = channels;
  n.groups = groups;
  n.w_f32 = w_dtype == GFD_DTYPE_F32;
  n.act = act;
  n.tile = c.tile;
  n.tiles = int(c.tiles);
  const void* ptrs[] = {x, y};
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    const int v = vector_of(channels / groups, sizeof(T), ptrs, 2, row_stride, ptr ? 0 : seg_stride);
    return with_vector(v, [&](auto w) {
      constexpr int V = decltype(w)::value;
      if constexpr (V * sizeof(T) <= 16) {
        int64_t blocks;
        return launch<T, V, false>(n, c, &blocks, static_cast<hipStream_t>(stream));
      } else {
        return GFD_ERR_UNSUPPORTED;
      }
    });
  });
}

gfd_status gfd_group_norm_bwd(const void* x, int dtype, int64_t segments, int64_t length,
                              const int64_t* ptr, int channels, int groups, int64_t row_stride,
                              int64_t seg_stride, const void* weight, const void* bias,
                              int w_dtype, int act, const double* stats, const void* grad_y,
                              void* grad_x, void* grad_weight, void* grad_bias, void* ws,
                              size_t ws_bytes, gfd_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  gfd_status st = check(x, dtype, segments, length, channels, groups, row_stride, seg_stride,
                        weight, bias, w_dtype, act);
  if (st != GFD_OK) return st;
  if (!aligned_to(grad_weight, dtype_size(w_dtype)) || !aligned_to(grad_bias, dtype_size(w_dtype)))
    return GFD_ERR_ARGUMENT;
  const bool rows = length > 0 && (ptr || segments > 0);
  if (rows && (!x || !grad_y || !grad_x || (!stats && segments > 0) ||
               !aligned_to(grad_y, dtype_size(dtype)) || !aligned_to(grad_x, dtype_size(dtype))))
    return GFD_ERR_ARGUMENT;
  Cut c = {};
  Norm n = {};
  int64_t blocks = 0;
  if (rows) {
    c = cut_of(segments, length, ptr != nullptr);
    if (!grid_ok(c, segments, ptr != nullptr)) return GFD_ERR_UNSUPPORTED;
    Carve cv(ws, ws_bytes);
    n.part = cv.take<double2>(size_t(c.slots + c.teams) * channels);
    n.mom = cv.take<double2>(c.tiled ? size_t(segments) * groups : 0);
    if (!cv.ok) return GFD_ERR_WORKSPACE;
    n.x = x;
    n.dy = grad_y;
    n.out = grad_x;
    n.ptr = ptr;
    n.segments = segments;
    n.length = length;
    n.row_stride = row_stride;
    n.seg_stride = seg_stride;
    n.w = weight;
    n.b = bias;
    n.stats = const_cast<double*>(stats);
    n.channels = channels;
    n.groups = groups;
    n.w_f32 = w_dtype == GFD_DTYPE_F32;
    n.act = act;
    n.tile = c.tile;
    n.tiles = int(c.tiles);
    n.part0 = int(c.slots);
    const void* ptrs[] = {x, grad_y, grad_x};
    st = with_dtype(dtype, [&](auto tag) {
      using T = decltype(tag);
      const int v = vector_of(channels / groups, sizeof(T), ptrs, 3, row_stride,
                              ptr ? 0 : seg_stride);
      return with_vector(v, [&](auto w) {
        constexpr int V = decltype(w)::value;
        if constexpr (V * sizeof(T) <= 16) {
          return launch<T, V, true>(n, c, &blocks, stream);
        } else {
          return GFD_ERR_UNSUPPORTED;
        }
      });
    });
    if (st != GFD_OK) return st;
  }
  if (!grad_weight && !grad_bias) return GFD_OK;
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    k_columns<T><<<(channels + 7) / 8, 256, 0, stream>>>(n.part, c.slots + blocks, channels,
                                                         w_dtype == GFD_DTYPE_F32, grad_weight,
                                                         grad_bias);
    GFD_LAUNCH_CHECK();
    return GFD_OK;
  });
}

}  // extern "C"
