// gfd_group_norm.hip -- group norm with an activation over node rows (channels
// last), forward and backward, dense or ragged segments of rows.
//
//   xhat = (x - mean_sg) rstd_sg,  z = xhat w + b,  y = act(z)
//   dz = dy act'(z),  A = mean_sg(w dz),  B = mean_sg(w dz xhat)
//   dx = rstd (w dz - A - xhat B),  dw = sum dz xhat,  db = sum dz
//
// Bound by memory: x in and y out (backward: x and dy in, dx out), with a few
// dozen operations an element.  A thread holds one vector of V channels of a
// row, V dividing the channels of a group, so that a vector lies in one group.
// Sums of a few rows of a thread are fp32, about its own first element (Shifted);
// everything that joins them is fp64, about an element of the group (base_of), so
// that a large mean costs nothing.  The column sums that blocks hand on for the
// weight and bias gradients are fp32: a rounding each, beside as many roundings of
// dz itself.
//   * A segment of one row (a node) is its group's lanes' own affair: they exchange
//     their sums and keep x in registers (k_rows); the backward finds the
//     statistics again.  203769 rows of 64 fp32 channels: forward 24 us, backward
//     30 us and 4 us for the weights (46, 59 and 12 us as teams with kept statistics).
//   * A short segment is normalised by one team of threads (k_team): its rows
//     are read twice, the second time from cache, in one launch.
//   * A long one is cut into tiles of rows: k_sums writes each tile's column
//     sums, k_join joins those of a segment and group in a fixed order, k_apply
//     writes the result.  8 x 16384 rows of 512 bf16 channels: forward 35 + 5 +
//     46 us, backward 55 + 6 + 67 us; what the two passes read and write takes 79
//     and 132 us at the rate of a copy.  A ragged segment is long when it has more rows than a
//     tile; then it holds the first or the last row of every tile that it
//     touches, so that a tile meets at most two of them and finds them by two
//     binary searches, however many segments there are.
//   * The weight and bias gradients are the column sums of all blocks and tiles,
//     added in a fixed order in k_join's launch.
#include "gfd_rowops.h"

using namespace gfd;

namespace {

constexpr int kMaxChannels = 2048;
constexpr int kTeamBlocks = 1024;  // backward: each leaves its column sums
constexpr int kMaxTeam = 1024;  // threads
constexpr int64_t kMaxTiled = 65535;  // dense segments in tiles: a launch's third dimension

struct Norm {
  const void* x;
  const void* dy;
  void* out;  // y or dx
  const int64_t* ptr;
  int64_t segments, length, row_stride, seg_stride;
  const void* w;
  const void* b;
  double* stats;   // [segments, groups, 2]
  double2* part;   // forward: column sums of x - c and (x - c)^2, c: base_of
  float2* grad_part;  // backward: of dz and dz xhat
  double2* mom;    // backward: A, B of a segment and group
  void* dw;        // backward, nullable
  void* db;
  double eps;
  int channels, groups, w_f32;
  int tile;        // rows of a tile; ragged segments up to it are short
  int tiles;       // of one segment (dense) or of all rows (ragged)
  int part0;       // first row of ``part`` that the teams write (backward)
  int cols, rows;  // threads over a row's vectors and over rows, powers of two
  int cols2, rows2;  // their logarithms
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

// the last segment that starts at or before row r, -1: none.  A whole wave: 64 probes at a time
__device__ __forceinline__ int64_t segment_of(const Norm& n, int64_t r) {
  const int lane = threadIdx.x & 63;
  int64_t lo = -1, hi = n.segments;  // lo starts at or before r, hi does not
  while (hi - lo > 1) {
    const int64_t step = (hi - lo - 1 + 63) / 64;
    const int64_t at = lo + 1 + lane * step;
    const int before = __popcll(__ballot(at < hi && ptr_at(n, at) <= r));  // the first ones
    const int64_t base = lo + 1;
    if (before > 0) lo = base + (before - 1) * step;
    if (base + before * step < hi) hi = base + before * step;
  }
  return lo;
}

struct Piece {
  int64_t seg, r0, r1;  // rows [r0, r1) of segment seg, none where r0 >= r1
  int64_t start;        // of the segment
};

// piece i (ragged: 0 or 1) of the long segments in tile t; its sums go to row 2 t + i (ragged) or
// seg * tiles + t of ``part``
__device__ __forceinline__ Piece piece_of(const Norm& n, int64_t t, int i) {
  const int64_t a = t * n.tile, e = a + n.tile < n.length ? a + n.tile : n.length;
  if (!n.ptr) {
    const int64_t s = blockIdx.z, base = s * n.length;
    return {s, base + a, base + e, base};
  }
  Piece p = {segment_of(n, i == 0 ? a : e - 1), 0, 0, 0};
  if (p.seg < 0) return p;
  segment_rows(n, p.seg, p.r0, p.r1);
  p.start = p.r0;
  // the second is the one that starts inside the tile
  if (p.r1 - p.r0 <= n.tile || (i == 1 && p.r0 <= a)) p.r1 = p.r0;
  p.r0 = p.r0 < a ? a : p.r0;
  p.r1 = p.r1 > e ? e : p.r1;
  return p;
}

template <typename T>
__device__ __forceinline__ const T* row_in(const Norm& n, const void* base, int64_t seg, int64_t r) {
  const T* p = static_cast<const T*>(base);
  return n.ptr ? p + r * n.row_stride
               : p + seg * n.seg_stride + (r - seg * n.length) * n.row_stride;
}

// what the sums of a segment (with rows, the first one ``start``) and the group whose first
// channel is ch are taken about in fp64: its first element.  However far from 0 the group lies,
// the sum of squares is at most its number of elements times the spread's, so that of 53 bits
// only as many go as that number has
template <typename T>
__device__ __forceinline__ T base_of(const Norm& n, int64_t seg, int64_t start, int ch) {
  return static_cast<const T*>(n.x)[(n.ptr ? start * n.row_stride : seg * n.seg_stride) + ch];
}

// ---------------------------------------------------------------------------
// element arithmetic
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float affine_at(const void* p, int f32, int c, float none) {
  if (!p) return none;
  return f32 ? static_cast<const float*>(p)[c] : to_f32(static_cast<const T*>(p)[c]);
}

// V of them
template <typename T, int V>
__device__ __forceinline__ void affine(const void* p, int f32, int c, float none, float (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = none;
  if (p && f32) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = static_cast<const float*>(p)[c + j];
  } else if (p) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = to_f32(static_cast<const T*>(p)[c + j]);
  }
}

__device__ __forceinline__ float exp_of(float v) { return __builtin_amdgcn_exp2f(v * 1.4426950408889634f); }

// a b - c, the product rounded like the one that c is a mean of: where c is that product alone, 0
// and not what its rounding left
__device__ __forceinline__ float less(float a, float b, float c) {
#pragma clang fp contract(off)
  return a * b - c;
}

// activation and, where d is not null, its derivative at z.  WIDE: of fp32 rows
template <int ACT, bool WIDE>
__device__ __forceinline__ float activate(float z, float* d) {
  switch (ACT) {
    case GFD_ACT_RELU:
      if (d) *d = z > 0.f ? 1.f : 0.f;
      return z > 0.f ? z : z != z ? z : 0.f;
    case GFD_ACT_SILU: {
      // (v_rcp_f32 and the exponential are within 2^-23 of themselves, as two roundings are)
      const float p = __builtin_amdgcn_rcpf(1.f + exp_of(-z));
      if (d) *d = p * (1.f + z * (1.f - p));
      return z * p;
    }
    case GFD_ACT_GELU: {
      const float e = exp_of(-0.5f * z * z);
      float p;  // Phi(z)
      if constexpr (WIDE) {
        p = fmaf(0.5f, erff(z * 0.70710678118654752f), 0.5f);
      } else {
        // Phi(-|z|) = e^(-z^2 / 2) times a polynomial in t = 1 / (1 + |z| / 4), fitted over 0 <=
        // |z| <= 14 so that Phi is within 4e-9 and its tail within 4e-5 of itself, a sixth of
        // half a step of fp16; its exponential is the derivative's too
        const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(z), 0.25f, 1.f));
        float q = fmaf(t, -0.0918481424f, 0.342620730f);
        q = fmaf(t, q, -0.268634528f);
        q = fmaf(t, q, 0.282492280f);
        q = fmaf(t, q, 0.0242558978f);
        q = fmaf(t, q, 0.112302706f);
        q = fmaf(t, q, 0.0988110527f) * t * e;
        p = z > 0.f ? 1.f - q : q;
      }
      if (d) *d = fmaf(z * e, 0.39894228040143268f, p);
      return z * p;
    }
    default:
      if (d) *d = 1.f;
      return z;
  }
}

// The columns of one vector in one segment: z = d A + B and xhat = d r - lr with d = x - hi, the
// mean split into hi + lo so that nothing is lost where it is far larger than the spread
template <typename T, int V, int ACT>
struct Columns {
  double mean, rstd;
  float hi, r, lr;
  float A[V], B[V];
  int c0;

  __device__ __forceinline__ void set(const Norm& n, int col, double m, double s) {
    mean = m;
    rstd = s;
    hi = float(m);
    r = float(s);
    lr = float((m - double(hi)) * s);
    c0 = col * V;
    affine<T, V>(n.w, n.w_f32, c0, 1.f, A);
    affine<T, V>(n.b, n.w_f32, c0, 0.f, B);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      B[j] = fmaf(-lr, A[j], B[j]);
      A[j] *= r;
    }
  }
  // z; where it is too near 0 for fp32 to tell relu's side, from fp64
  __device__ __forceinline__ float z(const Norm& n, float x, float d, int j) const {
    const float v = fmaf(d, A[j], B[j]);
    if (ACT == GFD_ACT_RELU && fabsf(v) <= 2e-6f * (fabsf(d * A[j]) + fabsf(B[j])))
      return float((double(x) - mean) * rstd * double(affine_at<T>(n.w, n.w_f32, c0 + j, 1.f)) +
                   double(affine_at<T>(n.b, n.w_f32, c0 + j, 0.f)));
    return v;
  }
  __device__ __forceinline__ Pack<T, V> forward(const Norm& n, const Raw<T, V>& x) const {
    Pack<T, V> y;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float v = x.at(j);
      y.v[j] = from_f32<T>(activate<ACT, sizeof(T) == 4>(z(n, v, v - hi, j), nullptr));
    }
    return y;
  }
  // dz and xhat
  __device__ __forceinline__ void slope(const Norm& n, const Raw<T, V>& x, const Raw<T, V>& dy,
                                        float (&dz)[V], float (&xh)[V]) const {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float v = x.at(j), d = v - hi;
      xh[j] = fmaf(d, r, -lr);
      float g;
      activate<ACT, sizeof(T) == 4>(z(n, v, d, j), &g);
      dz[j] = dy.at(j) * g;
    }
  }
  // ra, rb: r times the means of w dz and of w dz xhat
  __device__ __forceinline__ Pack<T, V> backward(const float (&dz)[V], const float (&xh)[V], float ra,
                                                 float rb) const {
    Pack<T, V> g;
#pragma unroll
    for (int j = 0; j < V; ++j) g.v[j] = from_f32<T>(fmaf(-xh[j], rb, less(A[j], dz[j], ra)));
    return g;
  }
};

// mean and 1 / sqrt(var + eps) from the sums of x - c and (x - c)^2 over n elements
__device__ __forceinline__ double2 moments_of(double s, double q, double n, double eps, double c) {
  const double mean = s / n;
  double var = q / n - mean * mean;
  if (var < 0.0) var = 0.0;
  return {c + mean, 1.0 / sqrt(var + eps)};
}

// the sum over the threads of a block that share a column (threadIdx.x % cols), in those of the
// first row: lanes of a wave by exchange, waves through LDS; a fixed order
__device__ __forceinline__ double2 sum_rows(double2 v, int cols, double2* red) {
  for (int d = cols; d < kWave; d <<= 1) {
    v.x += __shfl_xor(v.x, d);
    v.y += __shfl_xor(v.y, d);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int step = cols < kWave ? 1 : cols / kWave, width = cols < kWave ? cols : kWave;
  if (step * kWave < int(blockDim.x)) {
    __syncthreads();  // the last sum has been read
    if (lane < width) red[threadIdx.x] = v;
    __syncthreads();
    if (wave < step)
      for (int w = wave + step; w < int(blockDim.x) / kWave; w += step) {
        v.x += red[w * kWave + lane % width].x;
        v.y += red[w * kWave + lane % width].y;
      }
  }
  return v;
}

// A thread's sums of x and x^2 about c, in fp32 about its own first element k and, every few rows,
// into fp64 (a conversion to fp64 takes four times an fp32 operation): what rounding does to the
// deviations from k, however far k lies from 0, is not multiplied by it.  The squares of the k -
// mean of all threads are at most the sum of squares itself, so neither does an odd k cost digits.
struct Shifted {
  float k = 0.f, s = 0.f, q = 0.f;
  double a = 0.0, b = 0.0;
  int64_t n = 0;
  __device__ __forceinline__ void add(float x) {
    const float d = x - k;
    s += d;
    q = fmaf(d, d, q);
  }
  __device__ __forceinline__ void fold(int count) {
    a += double(s);
    b += double(q);
    s = q = 0.f;
    n += count;
  }
  // about c
  __device__ __forceinline__ double2 sums(double c) const {
    const double d = double(k) - c, m = double(n);
    return {fma(m, d, a), fma(d, fma(m, d, 2.0 * a), b)};
  }
};

// ---------------------------------------------------------------------------
// short segments: a team of cols x rows threads each
// ---------------------------------------------------------------------------
template <typename T, int V, int NC, bool BWD, int ACT>
__device__ __forceinline__ void do_team(const Norm& n, uint32_t block, uint32_t blocks, double2* lds) {
  double2* red = lds;                   // [blockDim]
  double2* col_sum = lds + blockDim.x;  // [teams][vecs]
  using P = Pack<T, V>;
  const int vecs = n.channels / V, gv = vecs / n.groups;
  const int size2 = n.cols2 + n.rows2, teams = blockDim.x >> size2;
  const int c = threadIdx.x & (n.cols - 1), tr = threadIdx.x >> n.cols2 & (n.rows - 1), team = threadIdx.x >> size2;
  double dw[NC][V] = {}, db[NC][V] = {};
  for (int64_t s0 = int64_t(block) * teams; s0 < n.segments; s0 += int64_t(blocks) * teams) {
    auto rows_of = [&](int64_t s, int64_t& r0, int64_t& r1) {
      r0 = r1 = 0;
      if (s < n.segments) {
        segment_rows(n, s, r0, r1);
        if (n.ptr && r1 - r0 > n.tile) r1 = r0;  // a long one: not here
      }
    };
    const int64_t seg = s0 + team;
    int64_t r0, r1;
    rows_of(seg, r0, r1);
    const bool any = r0 < r1;
    auto x_at = [&](int64_t r, int col) {
      Raw<T, V> v;
      v.read(row_in<T>(n, n.x, seg, r) + col * V);
      return v;
    };
    auto dy_at = [&](int64_t r, int col) {
      Raw<T, V> v;
      v.read(static_cast<const T*>(n.dy) + r * n.channels + col * V);
      return v;
    };
    // sums over the rows by column (f(k, col, a, b) adds a thread's), then of each group, handed
    // to done(a, b, its number of elements) and left at its first column
    auto reduce = [&](auto f, auto done) {
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const int col = c + k * n.cols;
        double a = 0.0, b = 0.0;
        if (col < vecs && any) f(k, col, a, b);
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
      for (int i = threadIdx.x; i < teams * n.groups; i += blockDim.x) {
        const int tm = i / n.groups, g = i - tm * n.groups;
        int64_t q0, q1;
        rows_of(s0 + tm, q0, q1);
        if (q0 >= q1) continue;
        double2* cs = col_sum + tm * vecs + g * gv;
        double a = 0.0, b = 0.0;
        for (int k = 0; k < gv; ++k) {
          a += cs[k].x;
          b += cs[k].y;
        }
        cs[0] = done(a, b, double(q1 - q0) * (n.channels / n.groups));
      }
      __syncthreads();
    };
    Columns<T, V, ACT> cols[NC];
    float ra[NC] = {}, rb[NC] = {};
    T base[NC];
    const bool kept = BWD && n.stats;  // the forward's moments; else they are found (again)
    if (!kept)
      reduce(
          [&](int k, int col, double& a, double& b) {
            Shifted t;
            base[k] = base_of<T>(n, seg, r0, col / gv * gv * V);
            for (int64_t r = r0 + tr; r < r1; r += n.rows) {
              const Raw<T, V> x = x_at(r, col);
              if (t.n == 0) t.k = x.at(0);
#pragma unroll
              for (int j = 0; j < V; ++j) t.add(x.at(j));
              t.fold(V);
            }
            const double2 v = t.sums(to_f32(base[k]));  // (converted here: nothing waits for it before)
            a = v.x;
            b = v.y;
          },
          [&](double a, double b, double count) { return moments_of(a, b, count, n.eps, 0.0); });
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int col = c + k * n.cols;
      if (col < vecs && any) {
        if (kept) {
          const double* st = n.stats + 2 * (seg * n.groups + col / gv);
          cols[k].set(n, col, st[0], st[1]);
        } else {
          const double2 m = col_sum[team * vecs + col / gv * gv];
          const double mean = double(to_f32(base[k])) + m.x;
          cols[k].set(n, col, mean, m.y);
          if (!BWD && n.stats && tr == 0 && col % gv == 0) {
            double* st = n.stats + 2 * (seg * n.groups + col / gv);
            st[0] = mean;
            st[1] = m.y;
          }
        }
      }
    }
    if (BWD) {
      if (!kept) __syncthreads();
      reduce(
          [&](int k, int col, double& a, double& b) {
            for (int64_t r = r0 + tr; r < r1; r += n.rows) {
              float dz[V], xh[V], sa = 0.f, sb = 0.f;
              cols[k].slope(n, x_at(r, col), dy_at(r, col), dz, xh);
#pragma unroll
              for (int j = 0; j < V; ++j) {
                const float f = dz[j] * xh[j];
                db[k][j] += double(dz[j]);
                dw[k][j] += double(f);
                sa = fmaf(cols[k].A[j], dz[j], sa);  // r times w
                sb = fmaf(cols[k].A[j], f, sb);
              }
              a += double(sa);
              b += double(sb);
            }
          },
          [](double a, double b, double count) { return double2{a / count, b / count}; });
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const int col = c + k * n.cols;
        if (col < vecs && any) {
          const double2 v = col_sum[team * vecs + col / gv * gv];
          ra[k] = float(v.x);
          rb[k] = float(v.y);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int col = c + k * n.cols;
      if (col < vecs && any) {
        for (int64_t r = r0 + tr; r < r1; r += n.rows) {
          P* out = reinterpret_cast<P*>(static_cast<T*>(n.out) + r * n.channels + col * V);
          if (BWD) {
            float dz[V], xh[V];
            cols[k].slope(n, x_at(r, col), dy_at(r, col), dz, xh);
            *out = cols[k].backward(dz, xh, ra[k], rb[k]);
          } else {
            *out = cols[k].forward(n, x_at(r, col));
          }
        }
      }
    }
    __syncthreads();
  }
  if (BWD) {  // this block's column sums of dz and dz xhat
    float2* part = n.grad_part + (int64_t(n.part0) + block) * n.channels;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int col = c + k * n.cols;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const double2 v = sum_rows({db[k][j], dw[k][j]}, n.cols, red);
        if (threadIdx.x < n.cols && col < vecs) part[col * V + j] = {float(v.x), float(v.y)};
      }
    }
  }
}

template <typename T, int V, int NC, bool BWD, int ACT>
__global__ void __launch_bounds__(kMaxTeam) k_team(const Norm n) {
  extern __shared__ double2 lds[];
  do_team<T, V, NC, BWD, ACT>(n, blockIdx.x, gridDim.x, lds);
}

// ---------------------------------------------------------------------------
// segments of one row whose groups are 1, 2, 4 .. 64 vectors: the lanes of a group exchange
// their sums, and x stays in registers
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;
constexpr int kRowBlocks = 2048;  // forward; backward: kTeamBlocks, each leaves its column sums

// the sum over the ``width`` (1, 2, 4 .. 64) neighbouring lanes of each such group, in all of them
__device__ __forceinline__ float near_sum(float v, int width) {
  auto from = [&](auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xF, 0xF, false));
  };
  using std::integral_constant;
  if (width > 1) v += from(integral_constant<int, 0xB1>{});   // lane ^ 1
  if (width > 2) v += from(integral_constant<int, 0x4E>{});   // lane ^ 2
  if (width > 4) v += from(integral_constant<int, 0x141>{});  // mirrored in 8: fours are equal by now
  if (width > 8) v += from(integral_constant<int, 0x140>{});  // mirrored in 16
  if (width > 16) v += __shfl_xor(v, 16);
  if (width > 32) v += __shfl_xor(v, 32);
  return v;
}

template <typename T, int V, bool BWD, int ACT>
__global__ void __launch_bounds__(kRowThreads) k_rows(const Norm n) {
  constexpr int R = BWD ? 2 : 4;  // rows in flight
  __shared__ double2 red[kRowThreads];
  const int vecs = n.channels / V, gv = vecs / n.groups;
  const int c = threadIdx.x & (n.cols - 1), sub = threadIdx.x >> n.cols2, rows = kRowThreads >> n.cols2;
  const int col = blockIdx.y * n.cols + c;
  const bool on = col < vecs;
  const float inv = 1.f / float(n.channels / n.groups);
  float w[V], b[V];
  affine<T, V>(n.w, n.w_f32, on ? col * V : 0, 1.f, w);
  affine<T, V>(n.b, n.w_f32, on ? col * V : 0, 0.f, b);
  double dw[V] = {}, db[V] = {};
  const int64_t step = int64_t(gridDim.x) * rows;
  const T* px = static_cast<const T*>(n.x) + col * V;
  const T* pd = static_cast<const T*>(n.dy) + col * V;
  T* po = static_cast<T*>(n.out) + col * V;
  for (int64_t r0 = int64_t(blockIdx.x) * rows + sub; r0 - sub < n.segments; r0 += R * step) {
    Raw<T, V> x[R], dy[R];
#pragma unroll
    for (int u = 0; u < R; ++u) {
      x[u] = dy[u] = Raw<T, V>{};
      if (on && r0 + u * step < n.segments) {
        x[u].read(px + (r0 + u * step) * n.seg_stride);
        if (BWD) dy[u].read(pd + (r0 + u * step) * n.channels);
      }
    }
    float e[V] = {}, f[V] = {};
#pragma unroll
    for (int u = 0; u < R; ++u) {
      // the mean in two steps: about a first one, which rounding leaves a little off, d is small
      float d[V], s = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) s += x[u].at(j);
      const float m = near_sum(s, gv) * inv;
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        d[j] = x[u].at(j) - m;
        s1 += d[j];
        s2 = fmaf(d[j], d[j], s2);
      }
      const float off = near_sum(s1, gv) * inv;
      const float var = fmaxf(fmaf(-off, off, near_sum(s2, gv) * inv), 0.f);
      // a row beyond the last, whose variance of 0 an eps of 0 leaves, adds 0 to the column sums
      const float r = BWD && r0 + u * step >= n.segments ? 0.f : rsqrtf(var + float(n.eps));
      const float lr = off * r;
      float xh[V], z[V];
      bool near = false;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        xh[j] = fmaf(d[j], r, -lr);
        z[j] = fmaf(xh[j], w[j], b[j]);
        if (ACT == GFD_ACT_RELU) near = near || fabsf(z[j]) <= 4e-6f * (fabsf(xh[j] * w[j]) + fabsf(b[j]));
      }
      if (ACT == GFD_ACT_RELU && __ballot(near)) {  // relu's side from fp64
        double ds = 0.0, dq = 0.0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const double t = double(x[u].at(j)) - double(m);
          ds += t;
          dq += t * t;
        }
        for (int k = 1; k < gv; k <<= 1) {
          ds += __shfl_xor(ds, k);
          dq += __shfl_xor(dq, k);
        }
        const double2 mm = moments_of(ds, dq, double(n.channels / n.groups), n.eps, double(m));
        if (near) {
#pragma unroll
          for (int j = 0; j < V; ++j)
            z[j] = float((double(x[u].at(j)) - mm.x) * mm.y * double(w[j]) + double(b[j]));
        }
      }
      Pack<T, V> o;
      if (BWD) {
        float dz[V], sa = 0.f, sb = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float g;
          activate<ACT, sizeof(T) == 4>(z[j], &g);
          dz[j] = dy[u].at(j) * g;
          const float wd = w[j] * dz[j];
          sa += wd;
          sb = fmaf(wd, xh[j], sb);
          e[j] += dz[j];
          f[j] = fmaf(dz[j], xh[j], f[j]);
        }
        const float ma = near_sum(sa, gv) * inv, mb = near_sum(sb, gv) * inv;
#pragma unroll
        for (int j = 0; j < V; ++j) o.v[j] = from_f32<T>(r * (less(w[j], dz[j], ma) - xh[j] * mb));
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) o.v[j] = from_f32<T>(activate<ACT, sizeof(T) == 4>(z[j], nullptr));
      }
      if (on && r0 + u * step < n.segments)
        *reinterpret_cast<Pack<T, V>*>(po + (r0 + u * step) * n.channels) = o;
    }
    if (BWD) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        db[j] += double(e[j]);
        dw[j] += double(f[j]);
      }
    }
  }
  if (BWD) {
    float2* part = n.grad_part + int64_t(blockIdx.x) * n.channels;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double2 v = sum_rows({db[j], dw[j]}, n.cols, red);
      if (threadIdx.x < n.cols && on) part[col * V + j] = {float(v.x), float(v.y)};
    }
  }
}

// ---------------------------------------------------------------------------
// long segments
// ---------------------------------------------------------------------------
constexpr int kTileThreads = 256;

// column sums of a tile: forward [slot][vecs] of x - c and (x - c)^2, backward [slot][channels] of
// dz and dz xhat; ragged tiles have two slots, an unused one is 0.  (These kernels are kept small:
// with indexed pieces, 64-bit divisions and more rows in flight the sums of 26 MB in 49 ragged
// segments took 22 us, so 11.  Of their waves' cycles there 37 to 59 % wait for memory, 12 to 26 %
// for an instruction, of whose fetches up to 1 % miss.)
template <typename T, int V, bool BWD, int ACT>
__device__ __forceinline__ void do_sums(const Norm& n, int64_t t, double2* red) {
  constexpr int S = BWD ? V : 1;
  constexpr int R = BWD ? 2 : 8;  // rows in flight
  const int vecs = n.channels / V, gv = vecs / n.groups;
  const int c = threadIdx.x & (n.cols - 1), tr = threadIdx.x >> n.cols2, rows = kTileThreads >> n.cols2;
  const int col = blockIdx.y * n.cols + c;
  const bool on = col < vecs;
#pragma unroll 1
  for (int i = 0; i < (n.ptr ? 2 : 1); ++i) {
    const Piece p = piece_of(n, t, i);
    double a[S] = {}, b[S] = {};
    if (on && p.r0 < p.r1) {
      Columns<T, V, ACT> k;
      if (BWD) {
        const double* st = n.stats + 2 * (p.seg * n.groups + col / gv);
        k.set(n, col, st[0], st[1]);
      }
      Shifted t1;
      float e[V] = {}, f[V] = {};  // of a few rows, in fp32
      int held = 0;
      auto fold = [&]() {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          a[j % S] += double(e[j]);
          b[j % S] += double(f[j]);
          e[j] = f[j] = 0.f;
        }
        held = 0;
      };
      const T* px = row_in<T>(n, n.x, p.seg, p.r0 + tr) + col * V;
      const T* pd = static_cast<const T*>(n.dy) + (p.r0 + tr) * n.channels + col * V;
      const int64_t xs = rows * n.row_stride, ds = int64_t(rows) * n.channels;
      int left = int(p.r1 - p.r0) - tr;
      if (!BWD && left > 0) {
        Raw<T, V> x;
        x.read(px);
        t1.k = x.at(0);
      }
#pragma unroll 1
      for (; left > 0; left -= R * rows) {
        Raw<T, V> x[R], dy[R];
#pragma unroll
        for (int u = 0; u < R; ++u) {
          x[u] = dy[u] = Raw<T, V>{};
          if (u * rows < left) {
            x[u].read(px + u * xs);
            if (BWD) dy[u].read(pd + u * ds);
          }
        }
        px += R * xs;
        pd += R * ds;
        if (BWD) {  // a row beyond the last adds 0 (dy is 0)
#pragma unroll
          for (int u = 0; u < R; ++u) {
            float dz[V], xh[V];
            k.slope(n, x[u], dy[u], dz, xh);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              e[j] += dz[j];
              f[j] = fmaf(dz[j], xh[j], f[j]);
            }
          }
          if ((held += R) >= 32) fold();
        } else {
#pragma unroll
          for (int u = 0; u < R; ++u)
            if (u * rows < left) {
#pragma unroll
              for (int j = 0; j < V; ++j) t1.add(x[u].at(j));
            }
          t1.fold(V * (left > (R - 1) * rows ? R : (left + rows - 1) / rows));
        }
      }
      if (BWD) {
        fold();
      } else {
        const double2 v = t1.sums(to_f32(base_of<T>(n, p.seg, p.start, col / gv * gv * V)));
        a[0] = v.x;
        b[0] = v.y;
      }
    }
    const int64_t slot = n.ptr ? 2 * t + i : int64_t(blockIdx.z) * n.tiles + t;
    const bool any = p.r0 < p.r1;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      double2 v = {a[j], b[j]};
      if (any) v = sum_rows(v, n.cols, red);
      if (tr == 0 && on) {
        if (BWD) n.grad_part[slot * n.channels + col * V + j] = {float(v.x), float(v.y)};
        else n.part[slot * vecs + col] = v;
      }
    }
  }
}

template <typename T, int V, bool BWD, int ACT>
__global__ void __launch_bounds__(kTileThreads) k_sums(const Norm n) {
  __shared__ double2 red[kTileThreads];
  do_sums<T, V, BWD, ACT>(n, blockIdx.x, red);
}

// both, of a ragged batch: the short segments in the first ``teams`` blocks, the tiles' sums in
// those behind them (one after the other they take 10 us longer, forward, and 14 us, backward)
template <typename T, int V, bool BWD, int ACT>
__global__ void __launch_bounds__(kTileThreads) k_team_sums(const Norm team, const Norm tile, uint32_t teams) {
  extern __shared__ double2 lds[];
  if (blockIdx.x < teams)
    do_team<T, V, 1, BWD, ACT>(team, blockIdx.x, teams, lds);
  else
    do_sums<T, V, BWD, ACT>(tile, blockIdx.x - teams, lds);
}

constexpr int kJoinThreads = 256;

// the weight and bias gradients of 4 channels: their column sums of all slots in a fixed order
template <typename T>
__device__ void join_columns(const Norm& n, int64_t slots, int c0, double2* red) {
  const int c = c0 + (threadIdx.x & 3);
  double2 s = {0.0, 0.0};
  if (c < n.channels) {
#pragma unroll 8
    for (int64_t i = threadIdx.x >> 2; i < slots; i += kJoinThreads / 4) {
      const float2 v = n.grad_part[i * n.channels + c];
      s.x += double(v.x);
      s.y += double(v.y);
    }
  }
  s = sum_rows(s, 4, red);
  if (threadIdx.x < 4 && c < n.channels) {
    if (n.db) {
      if (n.w_f32) static_cast<float*>(n.db)[c] = float(s.x);
      else static_cast<T*>(n.db)[c] = from_f32<T>(float(s.x));
    }
    if (n.dw) {
      if (n.w_f32) static_cast<float*>(n.dw)[c] = float(s.y);
      else static_cast<T*>(n.dw)[c] = from_f32<T>(float(s.y));
    }
  }
}

// a block for each long segment and group, its tiles' sums (blocks from 0 to jobs); behind them
// a block for every 4 channels of the weight and bias gradients.  BY_TILE: blocks of tiles in
// the place of segments, of which there are more; at most one long segment starts in a tile, and
// then the tile's last row is its
template <typename T, int V, bool BWD, bool BY_TILE>
__global__ void __launch_bounds__(kJoinThreads) k_join(const Norm n, int64_t jobs, int64_t slots) {
  __shared__ double2 red[kJoinThreads];
  if (BWD && int64_t(blockIdx.x) >= jobs) {
    join_columns<T>(n, slots, int(blockIdx.x - jobs) * 4, red);
    return;
  }
  const int vecs = n.channels / V, per = n.channels / n.groups;
  const int width = BWD ? n.channels : vecs, each = BWD ? per : vecs / n.groups;
  const uint32_t at = blockIdx.x / uint32_t(n.groups);
  const int g = int(blockIdx.x - at * n.groups);
  int64_t s = at, r0, r1, first, count;
  if (BY_TILE) {
    const int64_t a = int64_t(at) * n.tile, e = a + n.tile < n.length ? a + n.tile : n.length;
    s = segment_of(n, e - 1);
    if (s < 0 || ptr_at(n, s) < a) return;
  }
  segment_rows(n, s, r0, r1);
  if (n.ptr) {
    if (r1 - r0 <= n.tile) return;
    first = r0 / n.tile;
    count = (r1 - 1) / n.tile - first + 1;
  } else {
    first = s * n.tiles;
    count = n.tiles;
  }
  double2 v = {0.0, 0.0};
  // threads over the group's columns (a power of two of them), the others over the tiles
  int wide2 = 0;
  while ((1 << wide2) < each && (1 << wide2) < kJoinThreads) ++wide2;
  const int step = kJoinThreads >> wide2;
  // ragged: the second slot where the segment starts inside the tile
  using Part = std::conditional_t<BWD, float2, double2>;
  const Part* from = (BWD ? reinterpret_cast<const Part*>(n.grad_part) : reinterpret_cast<const Part*>(n.part)) +
                     (n.ptr ? 2 * first : first) * width + g * each;
  const int64_t pitch = n.ptr ? 2 * width : width;
  const bool inside = n.ptr && r0 > first * n.tile;
  for (int c = threadIdx.x & ((1 << wide2) - 1); c < each; c += 1 << wide2) {
    const double w = BWD ? double(affine_at<T>(n.w, n.w_f32, g * each + c, 1.f)) : 1.0;
    double2 s = {0.0, 0.0};
#pragma unroll 8
    for (int k = threadIdx.x >> wide2; k < int(count); k += step) {
      const Part q = from[k * pitch + (k == 0 && inside ? width : 0) + c];
      s.x += double(q.x);
      s.y += double(q.y);
    }
    v.x += w * s.x;
    v.y += w * s.y;
  }
  v = sum_rows(v, 1, red);
  if (threadIdx.x == 0) {
    const double total = double(r1 - r0) * per;
    const int64_t job = s * n.groups + g;
    if (BWD) {
      n.mom[job] = {v.x / total, v.y / total};
    } else {
      const double2 m = moments_of(v.x, v.y, total, n.eps, to_f32(base_of<T>(n, s, r0, g * per)));
      n.stats[2 * job] = m.x;
      n.stats[2 * job + 1] = m.y;
    }
  }
}

template <typename T, int V, bool BWD, int ACT>
__global__ void __launch_bounds__(kTileThreads) k_apply(const Norm n) {
  using P = Pack<T, V>;
  constexpr int R = 2;  // rows in flight
  const int vecs = n.channels / V, gv = vecs / n.groups;
  const int c = threadIdx.x & (n.cols - 1), tr = threadIdx.x >> n.cols2, rows = kTileThreads >> n.cols2;
  const int col = blockIdx.y * n.cols + c;
  const bool on = col < vecs;
  const int64_t t = blockIdx.x;
#pragma unroll 1
  for (int i = 0; i < (n.ptr ? 2 : 1); ++i) {
    const Piece p = piece_of(n, t, i);
    if (!on || p.r0 >= p.r1) continue;
    const int64_t job = p.seg * n.groups + col / gv;
    Columns<T, V, ACT> k;
    k.set(n, col, n.stats[2 * job], n.stats[2 * job + 1]);
    float ra = 0.f, rb = 0.f;
    if (BWD) {
      ra = float(n.mom[job].x * k.rstd);
      rb = float(n.mom[job].y * k.rstd);
    }
    const T* px = row_in<T>(n, n.x, p.seg, p.r0 + tr) + col * V;
    const int64_t at = (p.r0 + tr) * n.channels + col * V;
    const T* pd = static_cast<const T*>(n.dy) + at;
    T* po = static_cast<T*>(n.out) + at;
    const int64_t xs = rows * n.row_stride, ds = int64_t(rows) * n.channels;
#pragma unroll 1
    for (int left = int(p.r1 - p.r0) - tr; left > 0; left -= R * rows) {
      Raw<T, V> x[R], dy[R];
#pragma unroll
      for (int u = 0; u < R; ++u) {
        x[u] = dy[u] = Raw<T, V>{};
        if (u * rows < left) {
          x[u].read(px + u * xs);
          if (BWD) dy[u].read(pd + u * ds);
        }
      }
#pragma unroll
      for (int u = 0; u < R; ++u) {
        P o;
        if (BWD) {
          float dz[V], xh[V];
          k.slope(n, x[u], dy[u], dz, xh);
          o = k.backward(dz, xh, ra, rb);
        } else {
          o = k.forward(n, x[u]);
        }
        if (u * rows < left) *reinterpret_cast<P*>(po + u * ds) = o;
      }
      px += R * xs;
      pd += R * ds;
      po += R * ds;
    }
  }
  if (n.ptr && on) {  // the rows of no segment
    const int64_t a = t * n.tile, e = a + n.tile < n.length ? a + n.tile : n.length;
    const int64_t first = ptr_at(n, 0), last = ptr_at(n, n.segments);
    if (a < first || e > last)
      for (int64_t r = a + tr; r < e; r += rows)
        if (r < first || r >= last)
          *reinterpret_cast<P*>(static_cast<T*>(n.out) + r * n.channels + col * V) = P{};
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

// Dense segments of one team each, or tiles: by the vectors that a thread of a team has, which it
// passes one after the other, and by the segments, which have to fill the card.  64 bf16 channels,
// forward + backward, team and tiles: 64 x 64 17 and 21 us, 64 x 256 29 and 24, 256 x 256 32 and
// 35, 256 x 512 59 and 44, 512 x 64 20 and 34, 1100 x 256 68 and 85, 1100 x 4000 1172 and 917,
// 5000 x 4000 4487 and 3927; 256 channels: 256 x 64 32 and 47, 256 x 256 109 and 77, 3000 x 300
// 798 and 979, 2048 x 1000 1938 and 1810.
bool as_team(int64_t segments, int64_t length, int channels) {
  const int64_t each = length * channels / (4 * 256);
  const int64_t most = 4 + segments / 16;
  return each <= (most < 128 ? most : 128) || segments > kMaxTiled;
}

// how a call is cut; depends on shapes alone, so that the workspace query agrees with the call
struct Cut {
  bool team, tiled;
  int tile;
  int64_t tiles;   // of a segment (dense) or of all rows (ragged)
  int64_t slots;   // tile slots
  int64_t teams;   // upper bound of the team kernel's blocks
};

Cut cut_of(int64_t segments, int64_t length, bool ragged, int channels) {
  Cut c;
  // tiles: about 1024 of them, 32 to 512 rows (more dense segments than kMaxTiled have none)
  const int64_t rows = ragged ? length : segments <= kMaxTiled ? segments * length : 0;
  int64_t tile = rows < 512 * 1024 ? pow2_up((rows + 1023) / 1024) : 512;
  tile = tile < 32 ? 32 : tile;
  c.tile = int(tile);
  if (ragged) {
    c.team = c.tiled = true;
    c.tiles = (length + tile - 1) / tile;
    c.slots = 2 * c.tiles;
  } else {
    c.team = as_team(segments, length, channels);
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

// the widest vector, of at most 4, that divides a group's channels and that every row starts at
// (8 16-bit channels a thread cost more in registers than their wider access brings)
int vector_of(int64_t per_group, size_t size, const void* const* ptrs, int n, int64_t row_stride,
              int64_t seg_stride) {
  int v = 4;
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
    case 4: return f(std::integral_constant<int, 4>{});
    case 2: return f(std::integral_constant<int, 2>{});
    default: return f(std::integral_constant<int, 1>{});
  }
}

template <typename F>
gfd_status with_act(int act, F f) {
  switch (act) {
    case GFD_ACT_RELU: return f(std::integral_constant<int, GFD_ACT_RELU>{});
    case GFD_ACT_SILU: return f(std::integral_constant<int, GFD_ACT_SILU>{});
    case GFD_ACT_GELU: return f(std::integral_constant<int, GFD_ACT_GELU>{});
    default: return f(std::integral_constant<int, GFD_ACT_NONE>{});
  }
}

template <typename T, int V, bool BWD, int ACT>
gfd_status launch(Norm n, const Cut& c, hipStream_t stream) {
  const int vecs = n.channels / V;
  int64_t team_blocks = 0;
  bool summed = false;  // the tiles' sums
  const int gv = vecs / n.groups;
  if (!n.ptr && n.length == 1 && gv <= kWave && (gv & (gv - 1)) == 0) {
    n.cols = pow2_up(vecs < kWave ? vecs : kWave);
    n.cols2 = __builtin_ctz(n.cols);
    const int rows = kRowThreads / n.cols;
    const int64_t need = (n.segments + rows - 1) / rows, most = BWD ? c.teams : kRowBlocks;
    team_blocks = need < most ? need : most;
    k_rows<T, V, BWD, ACT><<<dim3(unsigned(team_blocks), unsigned((vecs + n.cols - 1) / n.cols)),
                             kRowThreads, 0, stream>>>(n);
    GFD_LAUNCH_CHECK();
  } else if (c.team && n.segments > 0) {
    const int nc = vecs > kMaxTeam ? 2 : 1;
    n.cols = pow2_up((vecs + nc - 1) / nc);
    const int block = n.cols > 256 ? n.cols : 256;
    // threads over the rows: as many as a segment has, of the mean length when ragged
    const int64_t mean = n.ptr ? (n.length + n.segments - 1) / n.segments : n.length;
    const int most = block / n.cols, want = pow2_up(mean < most ? (mean < 1 ? 1 : mean) : most);
    n.rows = want < most ? want : most;
    n.cols2 = __builtin_ctz(n.cols);
    n.rows2 = __builtin_ctz(n.rows);
    const int teams = block / (n.cols * n.rows);
    int64_t grid = (n.segments + teams - 1) / teams;
    // forward: a block each (1100 x 1000 in 1024 blocks: 107 us, in as many as there are 72 us)
    const int64_t most_blocks = BWD || n.ptr ? c.teams : int64_t(1) << 24;
    grid = grid < most_blocks ? grid : most_blocks;
    team_blocks = grid;
    const size_t lds = sizeof(double2) * (size_t(block) + size_t(teams) * vecs);
    if (c.tiled && block == kTileThreads && grid + c.tiles < (int64_t(1) << 31)) {
      Norm m = n;
      m.cols = pow2_up(vecs);
      m.cols2 = __builtin_ctz(m.cols);
      k_team_sums<T, V, BWD, ACT><<<unsigned(grid + c.tiles), block, lds, stream>>>(n, m, unsigned(grid));
      summed = true;
    } else if (nc == 1) {
      k_team<T, V, 1, BWD, ACT><<<int(grid), block, lds, stream>>>(n);
    } else if constexpr (V == 1) {  // more vectors than threads
      k_team<T, V, 2, BWD, ACT><<<int(grid), block, lds, stream>>>(n);
    }
    GFD_LAUNCH_CHECK();
  }
  if (c.tiled && c.slots > 0) {
    n.cols = pow2_up(vecs < kTileThreads ? vecs : kTileThreads);
    n.cols2 = __builtin_ctz(n.cols);
    // (dense segments are at most kMaxTiled here)
    const dim3 grid(unsigned(c.tiles), unsigned((vecs + n.cols - 1) / n.cols),
                    n.ptr ? 1u : unsigned(n.segments));
    if (!summed) k_sums<T, V, BWD, BWD ? ACT : GFD_ACT_NONE><<<grid, kTileThreads, 0, stream>>>(n);
    GFD_LAUNCH_CHECK();
    const bool by_tile = n.ptr && n.segments > c.tiles;
    const int64_t jobs = (by_tile ? c.tiles : n.segments) * n.groups;
    const int64_t columns = BWD && (n.dw || n.db) ? (n.channels + 3) / 4 : 0;
    const unsigned joins = unsigned(jobs + columns);
    if (joins > 0) {
      if (by_tile) k_join<T, V, BWD, true><<<joins, kJoinThreads, 0, stream>>>(n, jobs, c.slots + team_blocks);
      else k_join<T, V, BWD, false><<<joins, kJoinThreads, 0, stream>>>(n, jobs, c.slots + team_blocks);
    }
    GFD_LAUNCH_CHECK();
    k_apply<T, V, BWD, ACT><<<grid, kTileThreads, 0, stream>>>(n);
    GFD_LAUNCH_CHECK();
  } else if (BWD && (n.dw || n.db)) {
    k_join<T, V, BWD, false><<<(n.channels + 3) / 4, kJoinThreads, 0, stream>>>(n, 0, team_blocks);
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

// tiles, and the blocks of k_join and the sums that they add, are counted in 32 bits (groups are
// at most channels, dense tiled segments at most kMaxTiled)
bool grid_ok(const Cut& c, int channels) {
  return !c.tiled || c.tiles < (int64_t(1) << 31) / channels - 1;
}

}  // namespace

extern "C" {

size_t gfd_group_norm_workspace_size(int64_t segments, int64_t length, int ragged, int channels,
                                     int groups, int backward) {
  if (!shape_ok(segments, length, channels, groups) || channels > kMaxChannels) return 0;
  if (!ragged && (segments == 0 || length == 0)) return 0;
  const Cut c = cut_of(segments, length, ragged != 0, channels);
  Sizer z;
  if (backward) z.take<float2>(size_t(c.slots + c.teams) * channels);
  else z.take<double2>(size_t(c.slots) * channels);
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
  const Cut c = cut_of(segments, length, ptr != nullptr, channels);
  if (!grid_ok(c, channels)) return GFD_ERR_UNSUPPORTED;
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
  n.stats = !ptr && length == 1 ? nullptr
            : stats             ? stats
            : c.tiled           ? reinterpret_cast<double*>(n.mom)
                                : nullptr;
  n.eps = eps;
  n.channels = channels;
  n.groups = groups;
  n.w_f32 = w_dtype == GFD_DTYPE_F32;
  n.tile = c.tile;
  n.tiles = int(c.tiles);
  const void* ptrs[] = {x, y};
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    const int v = vector_of(channels / groups, sizeof(T), ptrs, 2, row_stride, ptr ? 0 : seg_stride);
    return with_vector(v, [&](auto w) {
      return with_act(act, [&](auto a) {
        return launch<T, decltype(w)::value, false, decltype(a)::value>(n, c, static_cast<hipStream_t>(stream));
      });
    });
  });
}

gfd_status gfd_group_norm_bwd(const void* x, int dtype, int64_t segments, int64_t length,
                              const int64_t* ptr, int channels, int groups, int64_t row_stride,
                              int64_t seg_stride, const void* weight, const void* bias,
                              int w_dtype, double eps, int act, const double* stats, const void* grad_y,
                              void* grad_x, void* grad_weight, void* grad_bias, void* ws,
                              size_t ws_bytes, gfd_stream_t stream_) {
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  gfd_status st = check(x, dtype, segments, length, channels, groups, row_stride, seg_stride,
                        weight, bias, w_dtype, act);
  if (st != GFD_OK) return st;
  if (!aligned_to(grad_weight, dtype_size(w_dtype)) || !aligned_to(grad_bias, dtype_size(w_dtype)))
    return GFD_ERR_ARGUMENT;
  if (!(eps >= 0.0)) return GFD_ERR_ARGUMENT;
  const bool rows = length > 0 && (ptr || segments > 0);
  if (rows && (!x || !grad_y || !grad_x || (!stats && segments > 0 && (ptr || length > 1)) ||
               !aligned_to(grad_y, dtype_size(dtype)) || !aligned_to(grad_x, dtype_size(dtype))))
    return GFD_ERR_ARGUMENT;
  if (!rows) {  // no row: gradients of 0
    if (!grad_weight && !grad_bias) return GFD_OK;
    Norm n = {};
    n.channels = channels;
    n.w_f32 = w_dtype == GFD_DTYPE_F32;
    n.dw = grad_weight;
    n.db = grad_bias;
    return with_dtype(dtype, [&](auto tag) {
      k_join<decltype(tag), 1, true, false><<<(channels + 3) / 4, kJoinThreads, 0, stream>>>(n, 0, 0);
      GFD_LAUNCH_CHECK();
      return GFD_OK;
    });
  }
  const Cut c = cut_of(segments, length, ptr != nullptr, channels);
  if (!grid_ok(c, channels)) return GFD_ERR_UNSUPPORTED;
  Carve cv(ws, ws_bytes);
  Norm n = {};
  n.grad_part = cv.take<float2>(size_t(c.slots + c.teams) * channels);
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
  // a row of its own: its statistics are found again, which is less than reading them
  n.stats = !ptr && length == 1 ? nullptr : const_cast<double*>(stats);
  n.eps = eps;
  n.dw = grad_weight;
  n.db = grad_bias;
  n.channels = channels;
  n.groups = groups;
  n.w_f32 = w_dtype == GFD_DTYPE_F32;
  n.tile = c.tile;
  n.tiles = int(c.tiles);
  n.part0 = int(c.slots);
  const void* ptrs[] = {x, grad_y, grad_x};
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    const int v = vector_of(channels / groups, sizeof(T), ptrs, 3, row_stride,
                            ptr ? 0 : seg_stride);
    return with_vector(v, [&](auto w) {
      return with_act(act, [&](auto a) {
        return launch<T, decltype(w)::value, true, decltype(a)::value>(n, c, stream);
      });
    });
  });
}

}  // extern "C"
