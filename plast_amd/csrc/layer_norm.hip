// layer_norm.hip — layer norm over the last axis and its gradients. For a row x of C elements:
//   mu = sum x / C,  r = 1 / sqrt(sum (x - mu)^2 / C + eps),  n = (x - mu) r,  y = n w + b,
//   dx = r (g - sum g / C - n sum (g n) / C) with g = dy w,
//   dw = sum over rows of dy n,  db = sum over rows of dy.
// The mean of fp32 sums is off by some 1e-7 of the largest |x|: a row far from zero loses digits of x - mu. So mu is
// corrected by the mean of the differences d = x - mu themselves, which are small, in the pass that sums their squares:
//   mu' = mu + m, m = sum d / C,  sum (x - mu')^2 = sum d^2 - C m^2.
//
// The memory bounds it: x read and y written, x and dy read and dx written. So rows are held in registers between their sums and
// their results, up to 32768 elements of fp32 and 65536 of 16 bits forward and 16384 backward, and workgroups go from row to row
// with the next rows on their way (forward with up to 16 columns a lane), as one row's reads, sums and stores one after the other
// leave the memory idle. A lane keeps its columns' sums for dw and db over all of its rows. us, and TB/s of what passes the L2 caches:
// forward [16384, 4096] in fp32 86, 6.3; in bf16 46, 5.9; backward in bf16 66, 6.4, and 5 to join the workgroups' sums; [30011, 333] in
// fp32 15, 5.5 and 30, 4.1, its rows off the 16-byte addresses and 84 of 128 units there. Backward of 8193 to 16384 elements, 16 columns a lane,
// is more than registers hold: 76 to 153 spill in fp32, 4 to 115 in 16 bits ([4096, 9000] in bf16 112, 32 at a copy's rate). Longer
// rows are read by a workgroup each (three times; backward once for the means and once by columns): backward [512, 20000] in fp16
// 9 + 18, and 4 to join.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "rows.hpp"

namespace plast {
namespace {

constexpr int kRowBlock = 256;  // lanes of a workgroup

// What a launch needs of its tensors. map: of x, of y or dy, and of dx.
struct NormArgs {
  const void *x, *dy;
  void *y, *dx;
  const float *w, *b;
  float *stats;     // [rows][2]: mu, r
  float *dw, *db;   // either may be null: not wanted
  uint32_t first_row, rows, width;  // first_row: of a launch, where one cannot hold all
  float eps;
  RowMap<3> map;
};

// Results are stored past the caches and operands read through them: what fits the last-level cache is there for the backward pass.
// us, that / operands past the caches too, before units were read without branches: forward [30011, 333] in fp32 19.7 / 24.0,
// [16384, 4096] 100 / 98, backward [512, 20000] in fp16 42 / 56; results through the caches: forward [16384, 4096] 103.
template <class T>
__device__ __forceinline__ void store_any(typename Unit<T>::floats f, T *p) {
  __builtin_nontemporal_store(__builtin_convertvector(f, typename Unit<T>::vec), reinterpret_cast<typename Unit<T>::any *>(p));
}

// A unit's elements from column j on, zeros behind the row's end.
template <class T>
__device__ __forceinline__ typename Unit<T>::vec load_raw(const T *row, uint32_t j, uint32_t width) {
  constexpr uint32_t E = Unit<T>::E;
  if (j + E <= width) return *reinterpret_cast<const typename Unit<T>::any *>(row + j);
  typename Unit<T>::vec v = T(0.0f);
  if (j >= width) return v;
#pragma unroll
  for (uint32_t e = 0; e < E; ++e)
    if (j + e < width) v[e] = row[j + e];
  return v;
}
// How a row's units lie that its lanes hold: kWhole, all of them whole; kInside, those that reach beyond the row's end moved back to
// lie before it, where their first elements are other units' too; kAny, for rows shorter than a unit. The first two read without
// branches, so that the loads of several rows are told apart while they are on their way: us, rows as in kAny / kInside, forward
// [8192, 5000] in fp32 100 / 79, backward [60000, 100] in fp16 37 / 18, [8192, 5001] in bf16 129 / 80.
enum Fit { kWhole, kInside, kAny };
template <Fit FIT, class T>
__device__ __forceinline__ uint32_t place(uint32_t j, uint32_t width) {
  return FIT == kInside && j + Unit<T>::E > width ? width - Unit<T>::E : j;
}
template <Fit FIT, class T>
__device__ __forceinline__ typename Unit<T>::vec load_held(const T *row, uint32_t j, uint32_t width) {
  if constexpr (FIT == kAny) return load_raw(row, j, width);
  else return *reinterpret_cast<const typename Unit<T>::any *>(row + place<FIT, T>(j, width));
}
// Whether element e of the unit at column j is in the row and no other unit's.
template <Fit FIT, class T>
__device__ __forceinline__ bool owns(uint32_t e, uint32_t j, uint32_t width) {
  return FIT == kWhole || (FIT == kAny ? j + e < width : place<FIT, T>(j, width) + e >= j);
}
// A unit's own elements, zeros for others.
template <Fit FIT, class T>
__device__ __forceinline__ typename Unit<T>::floats own(typename Unit<T>::floats f, uint32_t j, uint32_t width) {
#pragma unroll
  for (uint32_t e = 0; e < Unit<T>::E; ++e) f[e] = owns<FIT, T>(e, j, width) ? f[e] : 0.0f;
  return f;
}
template <class T>
__device__ __forceinline__ typename Unit<T>::floats load_cols(const T *row, uint32_t j, uint32_t width) {
  return to_floats<T>(load_raw(row, j, width));
}
template <class T>
__device__ __forceinline__ void store_cols(typename Unit<T>::floats f, T *row, uint32_t j, uint32_t width) {
  constexpr uint32_t E = Unit<T>::E;
  if (j + E <= width) {
    store_any<T>(f, row + j);
    return;
  }
  if (j >= width) return;
#pragma unroll
  for (uint32_t e = 0; e < E; ++e)
    if (j + e < width) row[j + e] = T(f[e]);
}
template <Fit FIT, class T>
__device__ __forceinline__ void store_held(typename Unit<T>::floats f, T *row, uint32_t j, uint32_t width) {
  if constexpr (FIT == kAny) {
    store_cols<T>(f, row, j, width);
  } else if (FIT == kWhole || j + Unit<T>::E <= width) {
    store_any<T>(f, row + j);
  } else if (j < width) {
    const uint32_t at = place<FIT, T>(j, width);
#pragma unroll
    for (uint32_t e = 0; e < Unit<T>::E; ++e)
      if (at + e >= j) row[at + e] = T(f[e]);
  }
}
// E columns of a weight or bias.
template <int E>
struct Cols {
  typedef float floats __attribute__((ext_vector_type(E)));
};
template <int E>
__device__ __forceinline__ typename Cols<E>::floats load_w(const float *w, uint32_t j, uint32_t width) {
  typename Cols<E>::floats f = 0.0f;
  if (j + E <= width) {
#pragma unroll
    for (int q = 0; q < E; q += 4) {
      const f4 v = *reinterpret_cast<const f4u *>(w + j + q);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[q + e] = v[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (j + e < width) f[e] = w[j + e];
  }
  return f;
}

// The sums of a and b over a workgroup of W waves, in every lane. `lds` holds 2 W floats that the call before did not use.
template <int W>
__device__ __forceinline__ void block_sums(float &a, float &b, float *lds) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    a += __shfl_xor(a, d);
    b += __shfl_xor(b, d);
  }
  if constexpr (W > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) lds[2 * wave] = a, lds[2 * wave + 1] = b;
    __syncthreads();
    a = lds[0], b = lds[1];
#pragma unroll
    for (int w = 1; w < W; ++w) a += lds[2 * w], b += lds[2 * w + 1];
  }
}

// The sums of a and b over the L lanes that share a row, in each of them. `lds` holds two floats a wave that the call before did
// not use.
template <int L>
__device__ __forceinline__ void row_sums(float &a, float &b, float *lds) {
#pragma unroll
  for (int d = (L < 64 ? L : 64) / 2; d >= 1; d >>= 1) {
    a += __shfl_xor(a, d);
    b += __shfl_xor(b, d);
  }
  if constexpr (L > 64) {
    constexpr int W = L / 64;
    const int wave = threadIdx.x >> 6, first = wave / W * W;
    if ((threadIdx.x & 63) == 0) lds[2 * wave] = a, lds[2 * wave + 1] = b;
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) a += lds[2 * (first + w)], b += lds[2 * (first + w) + 1];
  }
}
template <class F>
__device__ __forceinline__ float unit_sum(F f) {
  if constexpr (sizeof(F) == 32) return ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
  else return (f[0] + f[1]) + (f[2] + f[3]);
}

// ------------------------------------------------------------------------- rows in registers

// A row in U units of each of L lanes: read once, written once. Workgroups go from row to row (B / L of them at a time), the units of
// the next two on their way, the weight and the bias in registers; with more than 16 columns a lane a row each.
template <class T, int L, int U, Fit FIT>
__global__ __launch_bounds__(L > kRowBlock ? L : kRowBlock) void fwd_held_kernel(NormArgs A) {
  typedef typename Unit<T>::floats F;
  typedef typename Unit<T>::vec V;
  constexpr int E = Unit<T>::E, B = L > kRowBlock ? L : kRowBlock;
  constexpr bool HOLD = U * E <= 16;
  typedef typename Cols<E>::floats W;
  __shared__ float lds[2][2 * B / 64];
  const uint32_t lane = threadIdx.x % L, C = A.width, step = gridDim.x * (B / L);
  const uint64_t row0 = A.first_row + uint64_t(blockIdx.x) * (B / L) + threadIdx.x / L, end = uint64_t(A.first_row) + A.rows;
  if (row0 >= end) return;  // L lanes together, and all of them where they meet
  struct Row {
    int64_t y;
    V v[U];
  };
  const auto load = [&](Row &o, uint64_t row) {
    if (FIT != kAny) row = row < end ? row : end - 1;
    else if (row >= end) return;
    const RowAt<3> at = row_at(A.map, uint32_t(row));
    o.y = at.at[1];
#pragma unroll
    for (int u = 0; u < U; ++u) o.v[u] = load_held<FIT>(static_cast<const T *>(A.x) + at.at[0], (u * L + lane) * E, C);
  };
  W w[HOLD ? U : 1], b[HOLD ? U : 1];
  const float inv = 1.0f / float(C);
  const auto turn = [&](Row &o, uint64_t row) {
    F f[U];
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) f[u] = own<FIT, T>(to_floats<T>(o.v[u]), (u * L + lane) * E, C), s += unit_sum(f[u]);
    T *y = static_cast<T *>(A.y) + o.y;
    if constexpr (HOLD) load(o, row + 2 * uint64_t(step));
    row_sums<L>(s, q, lds[0]);
    float mu = s * inv;
    s = q = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const F d = own<FIT, T>(f[u] - mu, (u * L + lane) * E, C);
      s += unit_sum(d);
      q += unit_sum(d * d);
    }
    row_sums<L>(s, q, lds[1]);
    const float m = s * inv, var = __builtin_elementwise_maximum(q * inv - m * m, 0.0f);  // NaN stays
    mu += m;
    const float r = 1.0f / sqrtf(var + A.eps);
    if (lane == 0) {
      A.stats[2 * row] = mu;
      A.stats[2 * row + 1] = r;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t j = (u * L + lane) * E;
      W a, c;
      if constexpr (HOLD) a = w[u], c = b[u];
      else a = load_w<E>(A.w, place<FIT, T>(j, C), C), c = load_w<E>(A.b, place<FIT, T>(j, C), C);
      store_held<FIT, T>(__builtin_elementwise_fma((f[u] - mu) * r, a, c), y, j, C);
    }
  };
  Row one, two;
  load(one, row0);
  if constexpr (!HOLD) {  // a row each
    turn(one, row0);
    return;
  }
  load(two, row0 + step);
  if constexpr (HOLD) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t j = place<FIT, T>((u * L + lane) * E, C);
      w[u] = load_w<E>(A.w, j, C);
      b[u] = load_w<E>(A.b, j, C);
    }
  }
  for (uint64_t row = row0;; row += 2 * uint64_t(step)) {
    turn(one, row);
    if (row + step >= end) return;
    turn(two, row + step);
    if (row + 2 * uint64_t(step) >= end) return;
  }
}

// The gradients of rows held as above, but one or two on their way: a lane keeps the shares of dw and db of its columns in registers, the workgroup's rows are
// joined at the end, and its share goes to part[workgroup][2][C]. x and dy are read once.
template <int L>
constexpr int kBwdBlock = L > 512 ? L : 512;
template <class T, int L, int U, Fit FIT, bool ADD>
__global__ __launch_bounds__(kBwdBlock<L>) void bwd_held_kernel(NormArgs A, float *part) {
  typedef typename Unit<T>::floats F;
  typedef typename Unit<T>::vec V;
  constexpr int E = Unit<T>::E, R = kBwdBlock<L> / L;  // rows at a time
  // rows on their way, as many as registers hold: with 16 columns a lane [4096, 16384] in bf16 104 us with one, 153 with two
  constexpr uint32_t AHEAD = U * E > 8 ? 1 : 2;
  typedef typename Cols<E>::floats W;
  __shared__ float lds[2][2 * kBwdBlock<L> / 64];
  const uint32_t group = threadIdx.x / L, lane = threadIdx.x % L, C = A.width, step = gridDim.x * R;
  const T *x = static_cast<const T *>(A.x), *dy = static_cast<const T *>(A.dy);
  struct Row {
    int64_t dx;
    float mu, r;
    V f[U], g[U];
  };
  const auto load = [&](Row &o, uint64_t row) {
    if (FIT != kAny) {
      row = row < A.rows ? row : A.rows - 1;
    } else if (row >= A.rows) {
      o.mu = o.r = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) o.f[u] = o.g[u] = T(0.0f);
      return;
    }
    const RowAt<3> at = row_at(A.map, uint32_t(row));
    o.dx = at.at[2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      o.f[u] = load_held<FIT>(x + at.at[0], (u * L + lane) * E, C);
      o.g[u] = load_held<FIT>(dy + at.at[1], (u * L + lane) * E, C);
    }
    o.mu = A.stats[2 * row], o.r = A.stats[2 * row + 1];
  };
  W w[U], dw[U], db[U];
  const float inv = 1.0f / float(C);
  int buffer = 0;
  const auto turn = [&](Row &o, uint64_t row) {
    float s = 0.0f, q = 0.0f;
    F f[U], g[U];
    const float r = o.r;
    T *dx = static_cast<T *>(A.dx) + o.dx;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t j = (u * L + lane) * E;
      f[u] = own<FIT, T>((to_floats<T>(o.f[u]) - o.mu) * r, j, C);
      g[u] = own<FIT, T>(to_floats<T>(o.g[u]), j, C);
    }
    load(o, row + AHEAD * uint64_t(step));
    if (FIT != kAny && R > 1 && row >= A.rows) {  // a row behind the last
#pragma unroll
      for (int u = 0; u < U; ++u) g[u] = 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      dw[u] = __builtin_elementwise_fma(g[u], f[u], dw[u]);
      db[u] += g[u];
      g[u] *= w[u];
      s += unit_sum(g[u]);
      q += unit_sum(g[u] * f[u]);
    }
    if (!A.dx) return;
    row_sums<L>(s, q, lds[buffer]);
    buffer ^= 1;
    s *= inv, q *= inv;
    if (R > 1 && row >= A.rows) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t j = (u * L + lane) * E;
      F d = r * __builtin_elementwise_fma(f[u], F(-q), g[u] - s);
      if constexpr (ADD) d += to_floats<T>(load_held<FIT>(dx, j, C));
      store_held<FIT, T>(d, dx, j, C);
    }
  };
  Row one, two;
  load(one, blockIdx.x * R + group);
  if constexpr (AHEAD == 2) load(two, blockIdx.x * R + step + group);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    w[u] = load_w<E>(A.w, place<FIT, T>((u * L + lane) * E, C), C);
    dw[u] = db[u] = 0.0f;
  }
  // all of a workgroup's lanes take as many turns
  for (uint64_t first = blockIdx.x * R; first < A.rows; first += AHEAD * uint64_t(step)) {
    turn(one, first + group);
    if constexpr (AHEAD == 2)
      if (first + step < A.rows) turn(two, first + step + group);
  }
  if (!part) return;
  // the groups' shares, halves onto halves
  __shared__ float other[R > 1 ? (R / 2) * L * U * E : 1];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    W *mine = k ? db : dw;
#pragma unroll
    for (int h = R / 2; h >= 1; h /= 2) {
      __syncthreads();
      if (group >= uint32_t(h) && group < 2 * uint32_t(h)) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < E; ++e) other[(((group - h) * U + u) * E + e) * L + lane] = mine[u][e];
      }
      __syncthreads();
      if (group < uint32_t(h)) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < E; ++e) mine[u][e] += other[((group * U + u) * E + e) * L + lane];
      }
    }
    if (group == 0) {
      float *p = part + (uint64_t(blockIdx.x) * 2 + k) * C;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t j = (u * L + lane) * E;
          if (owns<FIT, T>(e, j, C)) p[place<FIT, T>(j, C) + e] = mine[u][e];
        }
    }
  }
}

// ------------------------------------------------------------------------- rows of any length

// A workgroup a row, read three times.
template <class T>
__global__ __launch_bounds__(kRowBlock) void fwd_long_kernel(NormArgs A) {
  typedef typename Unit<T>::floats F;
  constexpr uint32_t E = Unit<T>::E;
  __shared__ float lds[2][2 * kRowBlock / 64];
  const uint32_t row = A.first_row + blockIdx.x, C = A.width;
  const RowAt<3> at = row_at(A.map, row);
  const T *x = static_cast<const T *>(A.x) + at.at[0];
  T *y = static_cast<T *>(A.y) + at.at[1];
  const uint32_t step = kRowBlock * E, first = threadIdx.x * E;
  float s = 0.0f, q = 0.0f;
  for (uint32_t j = first; j < C; j += step) {
    const F f = load_cols<T>(x, j, C);
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) s += f[e];
  }
  block_sums<kRowBlock / 64>(s, q, lds[0]);
  float mu = s / float(C);
  s = q = 0.0f;
  for (uint32_t j = first; j < C; j += step) {
    const F f = load_cols<T>(x, j, C);
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
      const float d = j + e < C ? f[e] - mu : 0.0f;
      s += d;
      q = __builtin_fmaf(d, d, q);
    }
  }
  block_sums<kRowBlock / 64>(s, q, lds[1]);
  const float m = s / float(C);
  const float var = __builtin_elementwise_maximum(q / float(C) - m * m, 0.0f);  // NaN stays
  mu += m;
  const float r = 1.0f / sqrtf(var + A.eps);
  if (threadIdx.x == 0) {
    A.stats[2 * uint64_t(row)] = mu;
    A.stats[2 * uint64_t(row) + 1] = r;
  }
  for (uint32_t j = first; j < C; j += step) {
    F f = load_cols<T>(x, j, C);
    const typename Cols<E>::floats w = load_w<E>(A.w, j, C), b = load_w<E>(A.b, j, C);
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) f[e] = __builtin_fmaf((f[e] - mu) * r, w[e], b[e]);
    store_cols<T>(f, y, j, C);
  }
}

// The means of g and of g n of a row, [rows][2]: a workgroup a row.
template <class T>
__global__ __launch_bounds__(kRowBlock) void row_means_kernel(NormArgs A, float *means) {
  typedef typename Unit<T>::floats F;
  constexpr uint32_t E = Unit<T>::E;
  __shared__ float lds[2 * kRowBlock / 64];
  const uint32_t row = A.first_row + blockIdx.x, C = A.width;
  const RowAt<3> at = row_at(A.map, row);
  const T *x = static_cast<const T *>(A.x) + at.at[0], *dy = static_cast<const T *>(A.dy) + at.at[1];
  const float mu = A.stats[2 * uint64_t(row)], r = A.stats[2 * uint64_t(row) + 1];
  float s = 0.0f, q = 0.0f;
  for (uint32_t j = threadIdx.x * E; j < C; j += kRowBlock * E) {
    const F f = load_cols<T>(x, j, C), u = load_cols<T>(dy, j, C);
    const typename Cols<E>::floats w = load_w<E>(A.w, j, C);
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
      const float g = u[e] * w[e];  // 0 behind the end
      s += g;
      if (j + e < C) q = __builtin_fmaf(g, (f[e] - mu) * r, q);
    }
  }
  block_sums<kRowBlock / 64>(s, q, lds);
  if (threadIdx.x == 0) {
    means[2 * uint64_t(row)] = s / float(C);
    means[2 * uint64_t(row) + 1] = q / float(C);
  }
}

// Columns of some rows: a workgroup's lanes hold E columns each; blockIdx.x counts the blocks of columns of each piece of `per`
// rows. dx from the rows' means (null: not wanted), and the piece's share of dw and db to part[piece][2][C]. kColRows rows are read before the first of them is stored, as no load passes a store: backward of [512, 20000] in fp16 in all
// 32.4 us row by row, 30.4 with four, 29.9 with eight; with pieces of four rows 35.9.
constexpr uint32_t kColRows = 8;
template <class T, bool ADD, Fit FIT>
__global__ __launch_bounds__(kRowBlock) void columns_kernel(NormArgs A, const float *means, float *part, uint32_t blocks,
                                                            uint32_t per) {
  typedef typename Unit<T>::floats F;
  constexpr uint32_t E = Unit<T>::E;
  typedef typename Cols<E>::floats W;
  const uint32_t piece = blockIdx.x / blocks, C = A.width;
  const uint32_t j = ((blockIdx.x - piece * blocks) * kRowBlock + threadIdx.x) * E;
  if (j >= C) return;
  const W w = load_w<E>(A.w, place<FIT, T>(j, C), C);
  W dw = 0.0f, db = 0.0f;
  const uint32_t r0 = piece * per, r1 = r0 + per < A.rows ? r0 + per : A.rows;
  struct Row {
    int64_t dx;
    float mu, r, mg, mgn;
    typename Unit<T>::vec f, u;
  } o[kColRows];
  for (uint32_t row0 = r0; row0 < r1; row0 += kColRows) {
#pragma unroll
    for (uint32_t k = 0; k < kColRows; ++k) {
      const uint32_t row = row0 + k < r1 ? row0 + k : r1 - 1;
      const RowAt<3> at = row_at(A.map, row);
      o[k].dx = at.at[2];
      o[k].f = load_held<FIT>(static_cast<const T *>(A.x) + at.at[0], j, C);
      o[k].u = load_held<FIT>(static_cast<const T *>(A.dy) + at.at[1], j, C);
      o[k].mu = A.stats[2 * uint64_t(row)], o[k].r = A.stats[2 * uint64_t(row) + 1];
      if (means) o[k].mg = means[2 * uint64_t(row)], o[k].mgn = means[2 * uint64_t(row) + 1];
    }
#pragma unroll
    for (uint32_t k = 0; k < kColRows; ++k) {
      if (row0 + k >= r1) break;
      const F n = (to_floats<T>(o[k].f) - o[k].mu) * o[k].r, u = to_floats<T>(o[k].u);
      dw = __builtin_elementwise_fma(u, n, dw);
      db += u;
      if (means) {
        T *dx = static_cast<T *>(A.dx) + o[k].dx;
        F d = o[k].r * (__builtin_elementwise_fma(u, w, F(-o[k].mg)) - n * o[k].mgn);
        if constexpr (ADD) d += to_floats<T>(load_held<FIT>(dx, j, C));
        store_held<FIT, T>(d, dx, j, C);
      }
    }
  }
  if (part) {
    float *p = part + uint64_t(piece) * 2 * C + place<FIT, T>(j, C);
#pragma unroll
    for (uint32_t e = 0; e < E; ++e)
      if (owns<FIT, T>(e, j, C)) {
        p[e] = dw[e];
        p[C + e] = db[e];
      }
  }
}

// dw and db from the pieces' shares: 32 columns a workgroup, eight lanes a column, each every eighth piece.
constexpr uint32_t kFinCols = 32, kFinParts = 8;
template <bool ADD>
__global__ __launch_bounds__(kFinCols * kFinParts) void join_kernel(const float *part, uint32_t pieces, uint32_t width, uint64_t first,
                                                                    float *dw, float *db) {
  __shared__ float sums[kFinParts][kFinCols];
  const uint32_t col = threadIdx.x % kFinCols, k = threadIdx.x / kFinCols;
  const uint64_t i = first + uint64_t(blockIdx.x) * kFinCols + col, n = 2 * uint64_t(width);
  float *to = i < width ? dw : db;
  float s = 0.0f;
  if (i < n && to)
#pragma unroll 8
    for (uint32_t p = k; p < pieces; p += kFinParts) s += part[p * n + i];
  sums[k][col] = s;
  __syncthreads();
  if (k || i >= n || !to) return;
#pragma unroll
  for (uint32_t q = 1; q < kFinParts; ++q) s += sums[q][col];
  const uint64_t j = i < width ? i : i - width;
  to[j] = ADD ? to[j] + s : s;
}

// ------------------------------------------------------------------------- host

// Whether t lies like x: x's type and shape, a contiguous last axis.
bool like(const Tensor *t, const Tensor *x, uint64_t n) {
  const uint64_t last = x->ndim - 1;
  return t && t->device == GPU && t->dtype == x->dtype && same_shape(t, x) && (n == 0 || t->data) &&
         (x->shape[last] <= 1 || t->strides[last] == 1);
}

// Checks x, the weight, the bias, the statistics and eps; fills the row maps (of x, `second` and, where given, dx).
bool norm_args(NormArgs &A, const Tensor *const *inputs, const Tensor *second, const Tensor *dx, float eps,
               const char *where) {
  memset(&A, 0, sizeof A);
  const Tensor *x = inputs[0], *w = inputs[1], *b = inputs[2], *stats = inputs[3];
  if (!x || !w || !b || !stats || !second) {
    report_error(where, "a tensor is NULL");
    return false;
  }
  if (x->device != GPU || !is_float(x) || x->ndim < 1 || x->ndim > PLAST_MAX_NDIM) {
    report_error(where, "x must be a GPU tensor of FLOAT32, FLOAT16 or BFLOAT16 with a last axis");
    return false;
  }
  const uint64_t C = x->shape[x->ndim - 1], n = numel(x);
  // the elements of a row, and of the units that its last workgroup has beyond it, stay within 31 bits
  if (C < 1 || C > (uint64_t(1) << 31) - 65536) {
    report_error(where, "rows of %llu elements are not supported", (unsigned long long)C);
    return false;
  }
  const uint64_t N = n / C;
  if (N >= uint64_t(1) << 31) {
    report_error(where, "%llu rows are not supported", (unsigned long long)N);
    return false;
  }
  if (C > 1 && x->strides[x->ndim - 1] != 1) {
    report_error(where, "the last axis of x must be contiguous, not strided by %llu",
                 (unsigned long long)x->strides[x->ndim - 1]);
    return false;
  }
  if (n && !x->data) {
    report_error(where, "x has no data");
    return false;
  }
  if (!f32_vector(w, C) || !f32_vector(b, C)) {
    report_error(where, "weight and bias must be contiguous FLOAT32 GPU tensors of %llu elements", (unsigned long long)C);
    return false;
  }
  if (!f32_vector(stats, 2 * N)) {
    report_error(where, "stats must be a contiguous FLOAT32 GPU tensor of 2 N elements, N = %llu", (unsigned long long)N);
    return false;
  }
  if (!(eps > 0.0f && eps <= FLT_MAX)) {
    report_error(where, "eps must be finite and above 0, not %g", double(eps));
    return false;
  }
  A.x = x->data;
  A.w = static_cast<const float *>(w->data);
  A.b = static_cast<const float *>(b->data);
  A.stats = static_cast<float *>(stats->data);
  A.rows = uint32_t(N);
  A.width = uint32_t(C);
  A.eps = eps;
  Space s;
  s.rank = int(x->ndim) - 1;
  s.nops = 3;
  for (int d = 0; d < s.rank; ++d) {
    s.shape[d] = x->shape[d];
    s.st[0][d] = int64_t(x->strides[d]);
    s.st[1][d] = int64_t(second->strides[d]);
    s.st[2][d] = dx ? int64_t(dx->strides[d]) : 0;
  }
  if (!n) return true;
  collapse(s);
  A.map.rank = s.rank;
  for (int d = 0; d < s.rank; ++d) {
    A.map.ext[d] = MagicDiv::make(uint32_t(s.shape[d]));
    for (int k = 0; k < 3; ++k) A.map.st[k][d] = s.st[k][d];
  }
  return true;
}

// launch(args, workgroups) for parts of the rows that one grid holds, a workgroup of `threads` lanes for `per` rows.
template <class F>
void by_parts(const NormArgs &A, uint64_t per, uint64_t threads, F &&launch) {
  const uint64_t most = max_blocks(threads) * per;
  NormArgs part = A;
  for (uint64_t r = 0; r < A.rows; r += most) {
    part.first_row = uint32_t(r);
    part.rows = uint32_t(A.rows - r < most ? A.rows - r : most);
    launch(part, ceil_div(part.rows, per));
  }
}

// The shapes of rows that registers hold, lanes a row and units a lane, the first that holds a row taken; up to MOST units a lane, MOST1024
// of 1024 lanes.
struct Held {
  int lanes, units;
};
constexpr Held kHeld[] = {{16, 1},  {16, 2},  {16, 4},  {64, 2},   {64, 4},   {256, 1},  {256, 2},
                          {256, 4}, {512, 1}, {512, 2}, {1024, 1}, {1024, 2}, {1024, 4}, {1024, 8}};
constexpr int kHeldShapes = sizeof kHeld / sizeof *kHeld;
// Whether any row takes shape i: none before it holds as much.
template <int MOST, int MOST1024>
constexpr bool taken(int i) {
  const auto fits = [](Held h) { return h.units <= (h.lanes == 1024 ? MOST1024 : MOST); };
  for (int k = 0; k < i; ++k)
    if (fits(kHeld[k]) && kHeld[k].lanes * kHeld[k].units >= kHeld[i].lanes * kHeld[i].units) return false;
  return fits(kHeld[i]);
}
// f(lanes, units) for rows of `units` units; false for longer ones.
template <int MOST, int MOST1024, int I = 0, class F>
bool with_held(uint32_t units, F &&f) {
  using std::integral_constant;
  if constexpr (I < kHeldShapes) {
    if constexpr (taken<MOST, MOST1024>(I))
      if (units <= uint32_t(kHeld[I].lanes * kHeld[I].units)) {
        f(integral_constant<int, kHeld[I].lanes>{}, integral_constant<int, kHeld[I].units>{});
        return true;
      }
    return with_held<MOST, MOST1024, I + 1>(units, f);
  }
  return false;
}

// f(how a row's units lie that lanes hold in `UNITS` units).
template <class T, int UNITS, class F>
void with_fit(uint32_t width, F &&f) {
  using std::integral_constant;
  if (width == UNITS * Unit<T>::E) return f(integral_constant<Fit, kWhole>{});
  if constexpr (UNITS == 16)
    if (width < Unit<T>::E) return f(integral_constant<Fit, kAny>{});
  f(integral_constant<Fit, kInside>{});
}

// Workgroups of 256 lanes that go from row to row, for each CU: [16384, 4096] in bf16 51 us with four, 52 with eight, a row
// each 62.
constexpr uint64_t kFwdPerCu = 4;
template <class T>
void launch_forward(const NormArgs &A) {
  const bool held = with_held<16 / int(Unit<T>::E), 8>(ceil_div(A.width, Unit<T>::E), [&](auto lanes, auto units) {
    constexpr int L = decltype(lanes)::value, U = decltype(units)::value, B = L > kRowBlock ? L : kRowBlock;
    const auto launch = [](const NormArgs &part, unsigned blocks) {
      with_fit<T, L * U>(part.width, [&](auto fit) { fwd_held_kernel<T, L, U, decltype(fit)::value><<<blocks, B, 0, stream()>>>(part); });
    };
    if constexpr (U * int(Unit<T>::E) <= 16)  // goes from row to row
      launch(A, unsigned(std::min<uint64_t>(ceil_div(A.rows, B / L), uint64_t(num_cus()) * kFwdPerCu * kRowBlock / B)));
    else by_parts(A, B / L, B, launch);
  });
  if (!held)
    by_parts(A, 1, kRowBlock, [](const NormArgs &part, unsigned blocks) {
      fwd_long_kernel<T><<<blocks, kRowBlock, 0, stream()>>>(part);
    });
}

template <bool ADD>
void launch_join(const NormArgs &A, const float *part, uint64_t pieces) {
  // eight lanes a column: rows of 2^28 elements and more take several grids
  const uint64_t n = 2 * uint64_t(A.width), most = max_blocks(kFinCols * kFinParts) * kFinCols;
  for (uint64_t first = 0; first < n; first += most)
    join_kernel<ADD><<<ceil_div(std::min(n - first, most), kFinCols), kFinCols * kFinParts, 0, stream()>>>(
        part, uint32_t(pieces), A.width, first, A.dw, A.db);
}

// Rows that registers hold, eight columns a lane (16 in the longest rows): two workgroups of 512 lanes a CU.
template <class T, bool ADD>
bool launch_held_backward(const NormArgs &A, bool &held, const char *where) {
  bool ok = false;
  held = with_held<8 / int(Unit<T>::E), 16 / int(Unit<T>::E)>(ceil_div(A.width, Unit<T>::E), [&](auto lanes, auto units) {
    constexpr int L = decltype(lanes)::value, U = decltype(units)::value, R = kBwdBlock<L> / L;
    const uint64_t most = uint64_t(num_cus()) * (L > 512 ? 1 : 2);
    const uint64_t blocks = std::min<uint64_t>(most, ceil_div(A.rows, R));
    float *part = nullptr;
    if (A.dw || A.db) {
      part = static_cast<float *>(partials(blocks * 2 * A.width * sizeof(float), where));
      if (!part) return;
    }
    with_fit<T, L * U>(A.width, [&](auto fit) {
      bwd_held_kernel<T, L, U, decltype(fit)::value, ADD><<<unsigned(blocks), kBwdBlock<L>, 0, stream()>>>(A, part);
    });
    if (part) launch_join<ADD>(A, part, blocks);
    ok = true;
  });
  return ok;
}

// Rows of any length: their means, then columns of pieces of rows, then the pieces' sums.
template <class T, bool ADD>
bool launch_long_backward(const NormArgs &A, const char *where) {
  constexpr uint32_t E = Unit<T>::E;
  const uint32_t blocks = ceil_div(A.width, kRowBlock * E);
  // some 2048 workgroups, pieces of eight rows or more
  uint64_t pieces = 2048 / blocks;
  if (pieces < 1) pieces = 1;
  if (pieces > ceil_div(A.rows, 8)) pieces = ceil_div(A.rows, 8);
  const uint32_t per = ceil_div(A.rows, pieces);
  pieces = ceil_div(A.rows, per);
  const bool sums = A.dw || A.db;
  const uint64_t means_bytes = A.dx ? (8 * uint64_t(A.rows) + 255) / 256 * 256 : 0;
  const uint64_t part_bytes = sums ? pieces * 2 * A.width * sizeof(float) : 0;
  char *work = static_cast<char *>(partials(means_bytes + part_bytes, where));
  if (!work) return false;
  float *means = A.dx ? reinterpret_cast<float *>(work) : nullptr;
  float *part = sums ? reinterpret_cast<float *>(work + means_bytes) : nullptr;
  if (means)
    by_parts(A, 1, kRowBlock, [&](const NormArgs &p, unsigned n) {
      row_means_kernel<T><<<n, kRowBlock, 0, stream()>>>(p, means);
    });
  if (A.width % E == 0) columns_kernel<T, ADD, kWhole><<<unsigned(pieces * blocks), kRowBlock, 0, stream()>>>(A, means, part, blocks, per);
  else columns_kernel<T, ADD, kInside><<<unsigned(pieces * blocks), kRowBlock, 0, stream()>>>(A, means, part, blocks, per);
  if (sums) launch_join<ADD>(A, part, pieces);
  return true;
}

// A gradient that is wanted: null where it is not, reported where it does not fit.
bool vector_gradient(const Tensor *t, uint64_t n, float **out, const char *where) {
  *out = nullptr;
  if (!t->requires_grad) return true;
  if (!f32_vector(t->grad, n)) {
    report_error(where, "the gradients of weight and bias must be contiguous FLOAT32 GPU tensors of %llu elements",
                 (unsigned long long)n);
    return false;
  }
  *out = static_cast<float *>(t->grad->data);
  return true;
}

}  // namespace
}  // namespace plast

using namespace plast;

extern "C" {

void layer_norm_hip_forward(const Tensor **inputs, Tensor *output, KernelParams params) {
  const char *where = "layer_norm_hip_forward";
  NormArgs A;
  if (!norm_args(A, inputs, output, nullptr, params.fval, where)) return;
  if (!like(output, inputs[0], A.rows) || (numel(output) && overlapping(output))) {
    report_error(where, "the output must have x's type and shape, a contiguous last axis and rows that do not overlap");
    return;
  }
  const Tensor *x = inputs[0];
  for (uint64_t d = 0; A.rows && output->data == x->data && d + 1 < x->ndim; ++d)
    if (x->shape[d] > 1 && output->strides[d] != x->strides[d]) {
      report_error(where, "the output lies in the place of x with other strides");
      return;
    }
  const Operand y("the output", output), stats("stats", inputs[3]), at_x("x", x), w("weight", inputs[1]), b("bias", inputs[2]);
  if (output->data != x->data && !apart(y, {&at_x}, where)) return;
  if (!apart(y, {&w, &b, &stats}, where) || !apart(stats, {&at_x, &w, &b}, where)) return;
  if (A.rows == 0 || !ensure_init()) return;
  A.y = output->data;
  with_float_type(inputs[0]->dtype, [&](auto t) { launch_forward<decltype(t)>(A); });
  finish(where);
}

void layer_norm_hip_backward(Tensor **inputs, const Tensor *output, KernelParams params) {
  const char *where = "layer_norm_hip_backward";
  const Tensor *x = inputs[0], *dy = output ? output->grad : nullptr, *dx = x && x->requires_grad ? x->grad : nullptr;
  if (x && x->requires_grad && !dx) {
    report_error(where, "x requires a gradient but has none");
    return;
  }
  if (!dy) {
    report_error(where, "the output has no gradient");
    return;
  }
  NormArgs A;
  if (!norm_args(A, inputs, dy, dx, params.fval, where)) return;
  if (!like(dy, x, A.rows)) {
    report_error(where, "the output's gradient must have x's type and shape and a contiguous last axis");
    return;
  }
  if (dx && (!like(dx, x, A.rows) || (numel(dx) && overlapping(dx)))) {
    report_error(where, "the gradient of x must have x's type and shape, a contiguous last axis and rows that do not overlap");
    return;
  }
  if (dx && (dx->data == dy->data || dx->data == x->data) && A.rows) {
    report_error(where, "the gradient of x lies in the place of x or of the output's gradient");
    return;
  }
  if (!vector_gradient(inputs[1], A.width, &A.dw, where) || !vector_gradient(inputs[2], A.width, &A.db, where)) return;
  if (A.dw && A.dw == A.db) {
    report_error(where, "weight and bias have one gradient");
    return;
  }
  // what is joined last may lie where operands were
  const Operand to_x("the gradient of x", dx), to_w("the gradient of weight", A.dw ? inputs[1]->grad : nullptr),
      to_b("the gradient of bias", A.db ? inputs[2]->grad : nullptr);
  if (dx) {
    const Operand at_x("x", x), up("the output's gradient", dy), w("weight", inputs[1]), stats("stats", inputs[3]);
    if (!apart(to_x, {&at_x, &up, &w, &stats, &to_w, &to_b}, where)) return;
  }
  if (!apart(to_w, {&to_b}, where)) return;
  if (!dx && !A.dw && !A.db) return;
  const bool add = params.keepdim != 1;
  if (!ensure_init()) return;
  A.dy = dy->data;
  A.dx = dx ? dx->data : nullptr;
  if (A.rows == 0) {  // sums over no rows
    if (!add) {
      if (A.dw) zeros_hip(inputs[1]->grad, A.width);
      if (A.db) zeros_hip(inputs[2]->grad, A.width);
    }
    return;
  }
  bool ok = false;
  with_float_type(x->dtype, [&](auto t) {
    typedef decltype(t) T;
    bool held = false;
    ok = add ? launch_held_backward<T, true>(A, held, where) : launch_held_backward<T, false>(A, held, where);
    if (!held) ok = add ? launch_long_backward<T, true>(A, where) : launch_long_backward<T, false>(A, where);
  });
  if (ok) finish(where);
}

}  // extern "C"
