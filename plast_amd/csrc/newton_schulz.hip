// newton_schulz.hip — the Newton-Schulz orthogonalisation of a matrix, or of each of a stack, and the
// Muon optimizer step built on it.
//
// With G on the side with m <= n rows (transposed where it has more rows than columns) and
// X = G / (|G| + eps), Frobenius norm, each of `steps` iterations is
//   A = X X^T (m x m),  S = b A + c A A (m x m),  X = a X + S X (m x n).
// A and S are symmetric: their products compute the tiles on and below the diagonal and store each twice.
// Two steps can go at once: with P = a I + S the next X is P X and its A is P A P, all m x m, so that
//   PA = a A + S A,  A' = a PA + S PA,  S' = b A' + c A' A',  Q = a (S + S') + S' S,  X'' = a^2 X + Q X,
// polynomials of A that commute: their products are symmetric too. X is formed anew every second step, as an
// error of A' (of 2^-24, say) grows by a^2 with each step that goes without.
//
// The products run on the matrix units. fp32's own matrix instructions reach a sixteenth of fp16's rate,
// so every factor v is kept as two fp16, hi = round(v) and lo = round(v - hi), 22 significant bits (and a
// scale that keeps lo above fp16's subnormals), and a product is three
// instructions, hi hi + hi lo + lo hi, summed in fp32. What is left out, lo lo, is below 2^-22 of the
// product. The iteration in 64 bits is met to 4e-7 of the result at [256, 256] and [300, 800], where
// fp32 factors (24 bits, but one rounding per addition) meet it to 1.5e-6 and 1.8e-6.
//
// All three types take pairs: with hi alone a bf16 matrix is off by 1.4e-3 before its own rounding (a norm of
// 1.7e-3) instead of less than 1e-6.
//
// Layout of a factor ("lines"): each row is cut into lines of 128 bytes, a line holding 32 columns' hi
// and then their lo: what a workgroup's tile needs of a row in one step of the sum is one whole line, read
// from HBM, staged in LDS and read from there in 16-byte units. Rows and columns are padded with zeros to
// whole tiles, so the product has no bounds to check. Both operands of each product are read along their
// rows, X X^T, A A^T and S (X^T)^T, so X is kept in both orders; the update writes both.
#include <cfloat>
#include <cmath>
#include <cstdlib>
#include <mutex>
#include <unordered_set>
#include <vector>

#include "half_types.hpp"

namespace plast {
namespace {

constexpr int kNsBlock = 256;
constexpr uint32_t kNormParts = 1024;  // most workgroups that share a matrix's norm
constexpr int kPointers = 64;          // matrices of a launch that have pointers of their own

typedef f16_t h8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

// A stack of matrices with any strides, in elements.
struct Stack {
  const void *data;
  uint32_t rows, cols;
  int64_t sb, s0, s1;
};

struct MuonRule {
  float momentum, keep, scale;  // keep: 1 - lr decay; scale: lr sqrt(max(1, rows / cols))
  int nesterov;
};
// The matrices of a Muon launch.
struct MuonSet {
  const float *g[kPointers];
  float *m[kPointers], *p[kPointers];
  MuonRule rule;
};
__device__ __forceinline__ float muon_update(float g, float m, const MuonRule &R) {
  return R.nesterov ? (1.0f - R.momentum) * g + R.momentum * m : m;
}

// ------------------------------------------------------------------------- norms

__device__ __forceinline__ double block_sum(double s) {
  __shared__ double lds[kNsBlock / 64];
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  s = lds[0];
  for (int k = 1; k < kNsBlock / 64; ++k) s += lds[k];
  return s;
}

// |G|^2 in 64 bits, where neither the squares nor their sum overflow or vanish: one partial sum per
// workgroup.
template <class T>
__global__ __launch_bounds__(kNsBlock) void norm_kernel(Stack G, MagicDiv cols, double *part) {
  const T *g = static_cast<const T *>(G.data) + int64_t(blockIdx.y) * G.sb;
  const uint32_t n = G.rows * G.cols, stride = gridDim.x * kNsBlock;  // below 2^32
  double s = 0.0;
#pragma unroll 4
  for (uint64_t at = uint64_t(blockIdx.x) * kNsBlock + threadIdx.x; at < n; at += stride) {
    const uint32_t i = cols.div(uint32_t(at)), j = uint32_t(at) - i * G.cols;
    const double v = double(float(g[int64_t(i) * G.s0 + int64_t(j) * G.s1]));
    s += v * v;
  }
  s = block_sum(s);
  if (threadIdx.x == 0) part[uint64_t(blockIdx.y) * kNormParts + blockIdx.x] = s;
}

// Muon's: the momentum is updated in the same pass, and the norm is the update's.
__global__ __launch_bounds__(kNsBlock) void momentum_kernel(MuonSet S, uint64_t n, double *part) {
  const float *g = S.g[blockIdx.y];
  float *m = S.m[blockIdx.y];
  const bool vec = ((uintptr_t(g) | uintptr_t(m)) & 15) == 0;
  const uint64_t n4 = vec ? n / 4 : 0, at = uint64_t(blockIdx.x) * kNsBlock + threadIdx.x;
  const uint64_t stride = uint64_t(gridDim.x) * kNsBlock;
  const float b = S.rule.momentum;
  double s = 0.0;
  for (uint64_t i = at; i < n4; i += stride) {
    const f4 gi = reinterpret_cast<const f4 *>(g)[i];
    f4 v = reinterpret_cast<const f4 *>(m)[i];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      v[c] = b * v[c] + (1.0f - b) * gi[c];
      const double u = double(muon_update(gi[c], v[c], S.rule));
      s += u * u;
    }
    reinterpret_cast<f4 *>(m)[i] = v;
  }
  for (uint64_t i = n4 * 4 + at; i < n; i += stride) {
    const float v = b * m[i] + (1.0f - b) * g[i];
    m[i] = v;
    const double u = double(muon_update(g[i], v, S.rule));
    s += u * u;
  }
  s = block_sum(s);
  if (threadIdx.x == 0) part[uint64_t(blockIdx.y) * kNormParts + blockIdx.x] = s;
}

// |G| of matrix b from its partial sums, for a workgroup.
__device__ __forceinline__ double norm_of(const double *part, uint32_t b, uint32_t parts) {
  double s = 0.0;
  for (uint32_t k = threadIdx.x; k < parts; k += kNsBlock) s += part[uint64_t(b) * kNormParts + k];
  return sqrt(block_sum(s));
}

// ------------------------------------------------------------------------- lines

// The powers of two that X, A (and P A) and S (and Q) are kept times: 2^12, 2^12 and 2^11 for rules whose singular
// values stay around 1, less where the iteration leaves them no room below fp16's 65504.
struct Scales {
  float x, a, s;
};

// The power of two that one X is kept times: `scale` where |X| = |G| / (|G| + eps) is about 1. A smaller |G|
// leaves a small X, whose iterates grow by up to `growth` bits in all: it is raised by the bits that X lacks, less
// those that it may still grow by beyond the `room` above the largest iterate at `scale`.
__device__ __forceinline__ double scale_of_x(double norm, float eps, int growth, int room, float scale) {
  const double x = norm / (norm + double(eps));
  int lacks = x > 0.0 && x < 0.5 ? -ilogb(x) - 1 : 0;
  lacks = lacks > 110 ? 110 : lacks;
  const int grows = lacks < growth ? lacks : growth;
  return ldexp(double(scale), lacks - (grows > room ? grows - room : 0));
}

// A stack of factors in lines: `rows` padded rows of `pitch` bytes.
struct Lines {
  char *data;
  uint64_t pitch, next;  // bytes from one row, one matrix to the next
};
__device__ __forceinline__ char *line_at(const Lines &L, uint32_t b, uint32_t row, uint32_t col) {
  return L.data + b * L.next + row * L.pitch + (col >> 5) * 128 + (col & 31) * 2;
}
// Eight columns (a multiple of 8) of a row.
__device__ __forceinline__ void put8(char *at, const float *v) {
  h8 hi, lo;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    hi[e] = f16_t(v[e]);
    lo[e] = f16_t(v[e] - float(hi[e]));
  }
  *reinterpret_cast<h8 *>(at) = hi;
  *reinterpret_cast<h8 *>(at + 64) = lo;
}
__device__ __forceinline__ void get8(const char *at, float *v) {
  const h8 hi = *reinterpret_cast<const h8 *>(at), lo = *reinterpret_cast<const h8 *>(at + 64);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = float(hi[e]) + float(lo[e]);
}
__device__ __forceinline__ float get1(const char *at) {
  return float(*reinterpret_cast<const f16_t *>(at)) + float(*reinterpret_cast<const f16_t *>(at + 64));
}

// X and X^T in lines from the source, a 64x64 tile per workgroup, padding included.
template <class T, bool MUON>
__global__ __launch_bounds__(kNsBlock) void start_kernel(Stack G, MuonSet S, const double *part,
                                                         uint32_t parts, float eps, int growth,
                                                         int room, float base, Lines X, Lines XT, float *xscale) {
  __shared__ float tile[64][65];
  const uint32_t b = blockIdx.z, r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;  // of the source
  const bool tall = G.rows > G.cols;
  const T *g = static_cast<const T *>(G.data) + int64_t(b) * G.sb;
  float in[64 * 64 / kNsBlock];
#pragma unroll
  for (uint32_t k = 0; k < 64 * 64 / kNsBlock; ++k) {
    const uint32_t e = k * kNsBlock + threadIdx.x, r = r0 + e / 64, c = c0 + e % 64;
    in[k] = 0.0f;
    if (r < G.rows && c < G.cols) {
      if constexpr (MUON) {
        const uint64_t at = uint64_t(r) * G.cols + c;
        in[k] = muon_update(S.g[b][at], S.m[b][at], S.rule);
      } else {
        in[k] = float(g[int64_t(r) * G.s0 + int64_t(c) * G.s1]);
      }
    }
  }
  const double norm = norm_of(part, b, parts), sx = scale_of_x(norm, eps, growth, room, base);
  const double scale = sx / (norm + double(eps));
  if ((blockIdx.x | blockIdx.y | threadIdx.x) == 0) xscale[b] = float(sx);
#pragma unroll
  for (uint32_t k = 0; k < 64 * 64 / kNsBlock; ++k) {
    const uint32_t e = k * kNsBlock + threadIdx.x;
    tile[e / 64][e % 64] = float(double(in[k]) * scale);
  }
  __syncthreads();
  const Lines &R = tall ? XT : X, &C = tall ? X : XT;
  for (uint32_t e = threadIdx.x; e < 64 * 8; e += kNsBlock) {
    const uint32_t r = e / 8, c = e % 8 * 8;
    float v[8], w[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] = tile[r][c + k];
      w[k] = tile[c + k][r];
    }
    put8(line_at(R, b, r0 + r, c0 + c), v);
    put8(line_at(C, b, c0 + r, r0 + c), w);
  }
}

// ------------------------------------------------------------------------- products

// X X^T; a product of two symmetric factors that commute (polynomials of one matrix), with terms added; an
// update of X; the last one.
enum Mode { Gram, Square, Update, Final };

// Where the last step's result goes: out[b][i, j] (O), or p = p keep - scale * it.
struct Product {
  Lines u, v;         // the factors: C[i, j] = sum_k u[i, k] v[j, k]
  Lines in, in_t;     // the term added: A (Square), X and X^T (Update, Final)
  Lines out, out_t;   // the result and its transpose
  uint32_t lines;     // of a row
  uint32_t ti, tj;    // tiles
  uint32_t parts;     // the sum is cut into so many pieces
  float *partial;     // their sums, when there are several
  Lines in2;          // another term (Square), where it has data
  float alpha, beta, gamma;  // result = alpha sum + beta term + gamma term2, in the result's scale, of
  const float *xscale;  // X's scale in Gram and Final: by 1 / its square, 1 / it
  Stack o;
};

constexpr int kBlockLds = 32 * 33;  // floats of a block in LDS
// Orders a wave's writes to its part of LDS before its lanes' reads of each other's.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// Tile number -> (i, j): all of them, or those on and below the diagonal, row by row.
template <Mode M>
__device__ __forceinline__ void tile_at(uint32_t t, uint32_t ti, uint32_t &i, uint32_t &j) {
  if constexpr (M == Gram || M == Square) {
    i = uint32_t((sqrtf(8.0f * float(t) + 1.0f) - 1.0f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    j = t - i * (i + 1) / 2;
  } else {
    i = t % ti;
    j = t / ti;
  }
}

// What a block's result adds to its sums, a lane's sixteen columns of a row.
struct Term {
  h8 hi[2], lo[2];
};
template <Mode M>
__device__ __forceinline__ Term load_term(const Product &P, uint32_t b, uint32_t i0, uint32_t j0) {
  const uint32_t lane = threadIdx.x & 63, r = lane / 2, c = lane % 2 * 16;
  Term t;
  if constexpr (M != Gram) {
    const bool tall = M == Final && P.o.rows > P.o.cols;
    const char *at = tall ? line_at(P.in_t, b, j0 + r, i0 + c) : line_at(P.in, b, i0 + r, j0 + c);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      t.hi[h] = reinterpret_cast<const h8 *>(at)[h];
      t.lo[h] = reinterpret_cast<const h8 *>(at + 64)[h];
    }
  }
  return t;
}

// A block of 32x32 sums as the matrix unit leaves it: register r of a lane holds row
// 8 (r / 4) + 4 (lane / 32) + r % 4 of column lane % 32. It goes through LDS, so that rows and columns
// both leave as whole lines.
template <class T, Mode M, bool MUON>
__device__ __forceinline__ void put_block(const Product &P, const MuonSet &S, float *lds, f16v acc, const Term &term,
                                          uint32_t b, uint32_t i0, uint32_t j0, bool mirror) {
  const uint32_t lane = threadIdx.x & 63;
  float alpha = P.alpha, beta = P.beta;
  if constexpr (M == Gram || M == Final) {
    const float unscale = 1.0f / P.xscale[b];  // a power of two
    alpha *= unscale;
    if constexpr (M == Gram) alpha *= unscale;
    else beta *= unscale;
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) lds[(8 * (r / 4) + 4 * (lane / 32) + r % 4) * 33 + lane % 32] = alpha * acc[r];
  wave_sync();
  const uint32_t r = lane / 2, c = lane % 2 * 16;
  if constexpr (M == Final) {
    const bool tall = P.o.rows > P.o.cols;  // then the result is the transpose
    const uint32_t row0 = (tall ? j0 : i0) + lane / 32, col = (tall ? i0 : j0) + lane % 32;
    float old[16];  // the parameters, read together and ahead of their stores
    if constexpr (MUON) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t row = row0 + 2 * e;
        old[e] = row < P.o.rows && col < P.o.cols ? S.p[b][uint64_t(row) * P.o.cols + col] : 0.0f;
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
      lds[tall ? (c + e) * 33 + r : r * 33 + c + e] += beta * (float(term.hi[e / 8][e % 8]) + float(term.lo[e / 8][e % 8]));
    wave_sync();
    const uint32_t k = lane % 32;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const uint32_t q = 2 * e + lane / 32, row = row0 + 2 * e;
      const float v = tall ? lds[k * 33 + q] : lds[q * 33 + k];
      if (row >= P.o.rows || col >= P.o.cols) continue;
      if constexpr (MUON) {
        S.p[b][uint64_t(row) * P.o.cols + col] = old[e] * S.rule.keep - S.rule.scale * v;
      } else {
        T *o = static_cast<T *>(const_cast<void *>(P.o.data)) + int64_t(b) * P.o.sb;
        o[int64_t(row) * P.o.s0 + int64_t(col) * P.o.s1] = T(v);
      }
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[8], t[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = lds[r * 33 + c + 8 * h + e];
        if constexpr (M != Gram) v[e] = __builtin_fmaf(beta, float(term.hi[h][e]) + float(term.lo[h][e]), v[e]);
      }
      if (M == Square && P.in2.data) {
        get8(line_at(P.in2, b, i0 + r, j0 + c + 8 * h), t);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(P.gamma, t[e], v[e]);
      }
      put8(line_at(P.out, b, i0 + r, j0 + c + 8 * h), v);
      if (M != Gram && mirror)  // the transpose's lines take the same sums
#pragma unroll
        for (int e = 0; e < 8; ++e) lds[r * 33 + c + 8 * h + e] = v[e];
    }
    if (mirror) {
      wave_sync();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = lds[(c + 8 * h + e) * 33 + r];
        put8(line_at(P.out_t, b, j0 + r, i0 + c + 8 * h), v);
      }
    }
  }
  wave_sync();
}

// One tile of BM x BN outputs over one piece of the sum, by waves of WM x WN. Two stages of LDS: while
// the waves multiply one line of every row, the next lines are on their way into the other (loads straight
// to LDS; lane l of a load fills bytes 16 l of its 1 KiB, so a row's eight 16-byte units are permuted by
// choosing what each lane reads: unit c lies at c ^ (row / 2 % 8). A 16-byte LDS read is served for lanes 0-3, 12-15,
// 20-27 of a half wave together, then for the others, from 64 banks: this spreads either set over all of them). A ring of
// five half-line stages, four of them on their way, measured the same within 2%, with 4096 x 4096 in 4.28 ms and 4.30: the
// matrix units are at 1.1 PFLOP/s of fp16 in the long sums, what a large library product reaches here (4096 x 16384:
// 54-56% busy), and in the short ones wait for the tiles' ways out, when all workgroups store at once (24 x 1024 x
// 1024: 35% busy).
template <class T, Mode M, bool MUON, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN)) void product_kernel(Product P, MuonSet S) {
  constexpr int NW = (BM / WM) * (BN / WN), LOADS = (BM + BN) / 8 / NW, FA = WM / 32, FB = WN / 32;
  constexpr uint32_t STAGE = (BM + BN) * 128;
  constexpr uint32_t LDS = 2 * STAGE > NW * kBlockLds * 4 ? 2 * STAGE : NW * kBlockLds * 4;
  __shared__ __align__(128) char lds[LDS];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr bool sym = M == Gram || M == Square;
  const uint32_t tiles = sym ? P.ti * (P.ti + 1) / 2 : P.ti * P.tj;
  const uint32_t id = xcd_block(blockIdx.x, gridDim.x);
  const uint32_t b = id / (tiles * P.parts), rest = id - b * tiles * P.parts;
  const uint32_t part = rest / tiles, t = rest - part * tiles;
  uint32_t ti, tj;
  tile_at<M>(t, P.ti, ti, tj);
  const uint32_t first = uint32_t(uint64_t(P.lines) * part / P.parts);
  const uint32_t last = uint32_t(uint64_t(P.lines) * (part + 1) / P.parts);

  // this wave's loads: rows 8 q .. 8 q + 7 of the stage, q = wave * LOADS + k
  const char *src[LOADS];
#pragma unroll
  for (int k = 0; k < LOADS; ++k) {
    const uint32_t r = (wave * LOADS + k) * 8;
    const bool first_operand = r < BM;
    const Lines &L = first_operand ? P.u : P.v;
    const uint32_t row = (first_operand ? ti * BM + r : tj * BN + r - BM) + lane / 8;
    src[k] = L.data + b * L.next + row * L.pitch + ((lane % 8) ^ ((row >> 1) & 7)) * 16;
  }
  const auto fetch = [&](uint32_t line, uint32_t stage) {
#pragma unroll
    for (int k = 0; k < LOADS; ++k)
      __builtin_amdgcn_global_load_lds(
          reinterpret_cast<const __attribute__((address_space(1))) uint32_t *>(reinterpret_cast<uintptr_t>(src[k] + line * 128)),
          reinterpret_cast<__attribute__((address_space(3))) uint32_t *>(
              uint32_t(reinterpret_cast<uintptr_t>(&lds[stage * STAGE + (wave * LOADS + k) * 1024]))),
          16, 0, 0);
  };
  const uint32_t wi = wave / (BN / WN) * WM, wj = wave % (BN / WN) * WN;
  f16v acc[FA][FB];
#pragma unroll
  for (int a = 0; a < FA; ++a)
#pragma unroll
    for (int c = 0; c < FB; ++c)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][c][r] = 0.0f;

  fetch(first, 0);
  uint32_t stage = 0;
  for (uint32_t line = first; line < last; ++line, stage ^= 1) {
    __syncthreads();  // the line has arrived, and every wave is done with the other stage
    if (line + 1 < last) fetch(line + 1, stage ^ 1);
    const char *base = lds + stage * STAGE;
    const uint32_t row = lane % 32, key = (row >> 1) & 7;
#pragma unroll
    for (int g = 0; g < 2; ++g) {  // 16 columns each
      h8 ua[FA][2], vb[FB][2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint32_t unit = ((p * 4 + g * 2 + lane / 32) ^ key) * 16;
#pragma unroll
        for (int a = 0; a < FA; ++a)
          ua[a][p] = *reinterpret_cast<const h8 *>(base + (wi + a * 32 + row) * 128 + unit);
#pragma unroll
        for (int c = 0; c < FB; ++c)
          vb[c][p] = *reinterpret_cast<const h8 *>(base + (BM + wj + c * 32 + row) * 128 + unit);
      }
#pragma unroll
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int a = 0; a < FA; ++a)
#pragma unroll
          for (int c = 0; c < FB; ++c)
            acc[a][c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ua[a][q == 2], vb[c][q == 1], acc[a][c], 0, 0, 0);
    }
  }
  const uint32_t i0 = ti * BM + wi, j0 = tj * BN + wj;
  if (P.parts > 1) {
    f4 *to = reinterpret_cast<f4 *>(P.partial) +
             ((uint64_t(id) * NW + wave) * (FA * FB) * 4) * 64 + lane;
#pragma unroll
    for (int a = 0; a < FA; ++a)
#pragma unroll
      for (int c = 0; c < FB; ++c)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          to[((a * FB + c) * 4 + q) * 64] = f4{acc[a][c][4 * q], acc[a][c][4 * q + 1], acc[a][c][4 * q + 2],
                                               acc[a][c][4 * q + 3]};
    return;
  }
  Term next = load_term<M>(P, b, i0, j0);
  __syncthreads();  // the stages become the blocks' way out
  float *way = reinterpret_cast<float *>(lds) + wave * kBlockLds;
#pragma unroll
  for (int k = 0; k < FA * FB; ++k) {
    const Term term = next;  // the next block's is on its way while this one leaves
    if (k + 1 < FA * FB) next = load_term<M>(P, b, i0 + (k + 1) / FB * 32, j0 + (k + 1) % FB * 32);
    put_block<T, M, MUON>(P, S, way, acc[k / FB][k % FB], term, b, i0 + k / FB * 32, j0 + k % FB * 32, !sym || ti != tj);
  }
}

// Adds the pieces of a sum: a wave per 32x32 block.
template <class T, Mode M, bool MUON, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(kNsBlock) void join_kernel(Product P, MuonSet S) {
  constexpr int FA = WM / 32, FB = WN / 32, NB = (BM / 32) * (BN / 32);
  __shared__ float lds[kNsBlock / 64 * kBlockLds];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr bool sym = M == Gram || M == Square;
  const uint32_t tiles = sym ? P.ti * (P.ti + 1) / 2 : P.ti * P.tj;
  const uint32_t id = blockIdx.x * (kNsBlock / 64) + wave;  // NB is a multiple of 4: whole workgroups
  const uint32_t block = id % NB, tile = id / NB, b = tile / tiles, t = tile - b * tiles;
  uint32_t ti, tj;
  tile_at<M>(t, P.ti, ti, tj);
  const uint32_t w = block / (FA * FB), a = block % (FA * FB) / FB, c = block % FB;
  const uint32_t i0 = ti * BM + w / (BN / WN) * WM + a * 32, j0 = tj * BN + w % (BN / WN) * WN + c * 32;
  const Term term = load_term<M>(P, b, i0, j0);
  f16v acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
  for (uint32_t part = 0; part < P.parts; ++part) {
    const f4 *from = reinterpret_cast<const f4 *>(P.partial) +
                     ((uint64_t(b * P.parts + part) * tiles + t) * NB + block) * 4 * 64 + lane;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f4 v = from[q * 64];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[4 * q + e] += v[e];
    }
  }
  put_block<T, M, MUON>(P, S, lds + wave * kBlockLds, acc, term, b, i0, j0, !sym || ti != tj);
}

// Small products: a workgroup per 32x32 tile, whose eight waves each take a share of the sum straight from memory (a
// tile's factors are read by few others) and meet in LDS. One launch a product, where tiles of 64 leave most of the
// chip idle or need a second launch to join pieces.
constexpr int kSmallWaves = 8;
template <class T, Mode M, bool MUON>
__global__ __launch_bounds__(64 * kSmallWaves) void small_product_kernel(Product P, MuonSet S) {
  __shared__ float lds[kSmallWaves][kBlockLds];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr bool sym = M == Gram || M == Square;
  const uint32_t tiles = sym ? P.ti * (P.ti + 1) / 2 : P.ti * P.tj;
  const uint32_t b = blockIdx.x / tiles, t = blockIdx.x - b * tiles;
  uint32_t ti, tj;
  tile_at<M>(t, P.ti, ti, tj);
  const uint32_t first = P.lines * wave / kSmallWaves, last = P.lines * (wave + 1) / kSmallWaves;
  const uint32_t i0 = ti * 32, j0 = tj * 32;
  const char *u = P.u.data + b * P.u.next + (i0 + lane % 32) * P.u.pitch + lane / 32 * 16;
  const char *v = P.v.data + b * P.v.next + (j0 + lane % 32) * P.v.pitch + lane / 32 * 16;
  // the terms of the outputs that this thread will store, on their way while the sums are formed
  const uint32_t half = threadIdx.x / 256, e8 = threadIdx.x % 256;
  const bool stores = M == Final || (e8 < 128 && !(half && sym && ti == tj));
  const uint32_t row8 = (half ? j0 : i0) + e8 / 4, col8 = (half ? i0 : j0) + e8 % 4 * 8;
  float term[8];
  if constexpr (M == Square || M == Update)
    if (stores) get8(line_at(half ? P.in_t : P.in, b, row8, col8), term);
  f16v acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.0f;
  for (uint32_t line = first; line < last; ++line) {
    h8 ua[2][2], vb[2][2];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        ua[g][p] = *reinterpret_cast<const h8 *>(u + line * 128 + p * 64 + g * 32);
        vb[g][p] = *reinterpret_cast<const h8 *>(v + line * 128 + p * 64 + g * 32);
      }
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int q = 0; q < 3; ++q)
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ua[g][q == 2], vb[g][q == 1], acc, 0, 0, 0);
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) lds[wave][(8 * (r / 4) + 4 * (lane / 32) + r % 4) * 33 + lane % 32] = acc[r];
  __syncthreads();
  // the waves' sums, two outputs a thread, back into the first wave's tile
  for (uint32_t e = threadIdx.x; e < 32 * 32; e += 64 * kSmallWaves) {
    const uint32_t at = e / 32 * 33 + e % 32;
    float sum = lds[0][at];
#pragma unroll
    for (int w = 1; w < kSmallWaves; ++w) sum += lds[w][at];
    lds[0][at] = sum;
  }
  __syncthreads();
  // as put_block, an eighth of the tile a wave: rows by the first waves, the transpose's by the others
  float alpha = P.alpha, beta = P.beta;
  if constexpr (M == Gram || M == Final) {
    const float unscale = 1.0f / P.xscale[b];
    alpha *= unscale;
    if constexpr (M == Gram) alpha *= unscale;
    else beta *= unscale;
  }
  const float *tile = lds[0];
  if constexpr (M == Final) {
    const bool tall = P.o.rows > P.o.cols;
    for (uint32_t e = threadIdx.x; e < 32 * 32; e += 64 * kSmallWaves) {
      const uint32_t q = e / 32, k = e % 32;
      const uint32_t row = (tall ? j0 : i0) + q, col = (tall ? i0 : j0) + k;
      const char *at = tall ? line_at(P.in_t, b, j0 + q, i0 + k) : line_at(P.in, b, i0 + q, j0 + k);
      const float term = get1(at);
      const float r = __builtin_fmaf(beta, term, alpha * (tall ? tile[k * 33 + q] : tile[q * 33 + k]));
      if (row >= P.o.rows || col >= P.o.cols) continue;
      if constexpr (MUON) {
        float *p = S.p[b] + uint64_t(row) * P.o.cols + col;
        *p = *p * S.rule.keep - S.rule.scale * r;
      } else {
        T *o = static_cast<T *>(const_cast<void *>(P.o.data)) + int64_t(b) * P.o.sb;
        o[int64_t(row) * P.o.s0 + int64_t(col) * P.o.s1] = T(r);
      }
    }
  } else {
    if (!stores) return;
    const uint32_t r = e8 / 4, c = e8 % 4 * 8;
    float w[8], x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      w[k] = alpha * (half ? tile[(c + k) * 33 + r] : tile[r * 33 + c + k]);
      if constexpr (M != Gram) w[k] = __builtin_fmaf(beta, term[k], w[k]);
    }
    if (M == Square && P.in2.data) {
      get8(line_at(P.in2, b, row8, col8), x);
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = __builtin_fmaf(P.gamma, x[k], w[k]);
    }
    put8(line_at(half ? P.out_t : P.out, b, row8, col8), w);
  }
}

// No steps: the result is X.
template <class T, bool MUON>
__global__ __launch_bounds__(kNsBlock) void copy_out_kernel(Lines X, Lines XT, const float *xscale, Stack O,
                                                            MuonSet S) {
  const uint32_t b = blockIdx.z, i = blockIdx.y, j = blockIdx.x * kNsBlock + threadIdx.x;
  if (j >= O.cols) return;
  const char *at = line_at(O.rows > O.cols ? XT : X, b, i, j);
  const float v = get1(at) / xscale[b];
  if constexpr (MUON) {
    float *p = S.p[b] + uint64_t(i) * O.cols + j;
    *p = *p * S.rule.keep - S.rule.scale * v;
  } else {
    T *o = static_cast<T *>(const_cast<void *>(O.data)) + int64_t(b) * O.sb;
    o[int64_t(i) * O.s0 + int64_t(j) * O.s1] = T(v);
  }
}

// ------------------------------------------------------------------------- host

// How a product runs: its tiles, and the pieces its sums are cut into.
struct Tiling {
  uint32_t tile, parts;
};
// How a shape runs.
struct Plan {
  uint32_t m, n, mp, np;  // extents, and padded to whole tiles
  Tiling gram, square, update;
  bool pairs;       // steps go by pairs
  Scales scale;
  int growth, room;  // of X
};

// The pieces that leave the fewest rounds of `slots` workgroups, each a share of the sum. In lines' time, a round
// costs four beside its lines, and cutting the launch that joins the pieces, twelve (four of 256 wide tiles' longer
// ones), and eight per round of pieces
// (256 x 256 in 64 wide tiles without that: 177 us instead of 128; 6 x 1001 x 2605 in 128 wide ones 1216 and 1132).
uint32_t pieces(uint64_t tiles, uint32_t lines, uint64_t slots, double join) {
  uint32_t best = 1;
  double least = 1e300;
  for (uint32_t s = 1; s <= 16 && s <= lines; ++s) {
    const double rounds = double((tiles * s + slots - 1) / slots);
    const double t = rounds * (double(lines) / s + 4.0) + (s > 1 ? join + 8.0 * s * double(tiles) / double(slots) : 0.0);
    if (t < least * 0.98) {
      least = t;
      best = s;
    }
  }
  return best;
}

// Tiles of 64 and below: sums of up to 32 lines over up to 512 tiles of 32 go to the small products (256 x 256:
// 88 us instead of 128, 512 x 512 130 and 185; but 64 x 8000, 250 lines, 354 and 149, 20 x 300 x 300, 1100 tiles, 318
// and 181).
Tiling tiling(uint32_t tile, uint32_t rows, uint32_t cols, bool sym, uint64_t count, uint32_t lines) {
  const auto tiles = [&](uint64_t t) { return (sym ? rows / t * (rows / t + 1) / 2 : rows / t * (cols / t)) * count; };
  if (tile == 64 && lines <= 32 && tiles(32) <= 512) return {32, 1};
  return {tile, pieces(tiles(tile), lines, uint64_t(num_cus()) * (tile == 256 ? 1 : 2), tile == 256 ? 4.0 : 12.0)};
}

uint32_t round_up(uint32_t v, uint32_t to) { return (v + to - 1) / to * to; }

// The rule followed for singular values in [0, 1]: the scales that give each factor room, and whether two steps'
// factor, P' P - a^2, has room at the scale of S; `most` is the largest singular value met, `growth` the bits by
// which any grows at most, `room` those between `most` at its scale and fp16's range.
struct RuleRange {
  Scales scale;
  bool pairs;
  double most;
  int growth, room;
};
RuleRange follow(const NewtonSchulz &r) {
  double x = 1.0, a = 1.0, s = 0.0, q = 0.0, ratio = 1.0;
  for (int i = 1; i <= r.steps; ++i) ratio = std::fmax(ratio, std::pow(std::fabs(double(r.a)), i));  // towards 0
  for (int k = 0; k <= 4096; ++k) {
    const double from = double(k) / 4096.0;
    double v = from, before = 0.0;
    for (int i = 0; i < r.steps; ++i) {
      const double l = v * v, p = r.a + r.b * l + r.c * l * l;
      a = std::fmax(a, std::fmax(l, std::fabs(p * l)));
      s = std::fmax(s, std::fabs(r.b * l + r.c * l * l));
      if (i % 2) q = std::fmax(q, std::fabs(before * p - double(r.a) * r.a));
      before = p;
      v *= p;
      x = std::fmax(x, std::fabs(v));
      if (k) ratio = std::fmax(ratio, std::fabs(v) / from);
    }
  }
  const auto fit = [](double most, int bits) {
    while (bits > -100 && !(std::ldexp(most, bits) <= 32768.0)) --bits;
    return float(std::ldexp(1.0, bits));
  };
  const Scales to{fit(x, 12), fit(a, 12), fit(s, 11)};
  const double growth = std::ceil(std::log2(ratio));
  const double room = std::floor(std::log2(64000.0 / (x * to.x)));
  return RuleRange{to, q * to.s <= 32768.0, x, int(growth < 110.0 ? growth : 110.0), int(room > 0.0 ? room : 0.0)};
}
// The same, worked out once for each of the last eight rules (0.1 ms on the host at 5 steps, 30 ms at 1000).
RuleRange range_of(const NewtonSchulz &r) {
  constexpr int kRules = 8;
  static std::mutex mu;
  static NewtonSchulz rules[kRules];
  static RuleRange ranges[kRules];
  static int known = 0, next = 0;
  std::lock_guard<std::mutex> lk(mu);
  for (int k = 0; k < known; ++k)
    if (memcmp(&rules[k], &r, sizeof r) == 0) return ranges[k];
  const int at = next;
  rules[at] = r;
  ranges[at] = follow(r);
  next = (next + 1) % kRules;
  known = known < kRules ? known + 1 : kRules;
  return ranges[at];
}

Plan make_plan(uint32_t rows, uint32_t cols, uint64_t count, const NewtonSchulz &rule) {
  Plan p;
  p.m = rows < cols ? rows : cols;
  p.n = rows < cols ? cols : rows;
  // 256 wide tiles read each factor least often, 128 wide ones leave fewer workgroups without work: 4096 x 4096 4.39
  // and 4.83 ms, 2304 x 4608 1.45 and 1.49, 2048 x 2048 909 and 839 us, 24 x 1024 x 1024 2.31 and 2.25 ms. They pay where
  // they pad m by no more than 3% beyond the others (5200 x 5200, 2.4%: 8.37 and 9.19 ms; 2049 x 4200, 5.9%: 1.41 and 1.21,
  // 3100 x 6200, 4%: 3.68 and 3.27). 64 wide ones go on with that: 1024 x 1024 262 us (128: 324), 512 x 4096 246 (321),
  // 2048 x 2048 913.
  const uint64_t work = uint64_t(p.m) * p.n * count;
  const bool widest = p.m > 2048 && work >= uint64_t(1) << 23 && round_up(p.m, 256) * 100 <= round_up(p.m, 128) * 103;
  const uint32_t tile = widest ? 256 : p.m > 128 && work >= uint64_t(3) << 20 ? 128 : 64;
  // Two steps at once cost three more m x m products and one product of X X^T and one update of X less: 1.5 m^2 n
  // multiplications less for 1.5 m^3 more, and one launch more (4096 x 16384: 13.6 -> 10.4 ms, 6 x 2605 x 1001 in fp32 1.34 ->
  // 1.18; under 2^30 the launch costs more).
  const RuleRange range = range_of(rule);
  p.scale = range.scale;
  p.growth = range.growth;
  p.room = range.room;
  p.pairs = range.pairs && rule.steps >= 2 && uint64_t(p.m) * p.m * (p.n - p.m) * count >= uint64_t(1) << 30;
  p.mp = round_up(p.m, tile);
  p.np = round_up(p.n, tile);
  p.gram = tiling(tile, p.mp, p.mp, true, count, p.np / 32);
  p.square = tiling(tile, p.mp, p.mp, true, count, p.mp / 32);
  p.update = tiling(tile, p.mp, p.np, false, count, p.mp / 32);
  return p;
}

// Bytes of a workspace for `count` matrices: norms, X and X^T twice, A and S, and the pieces' sums.
uint64_t ns_bytes(const Plan &p, uint64_t count) {
  uint64_t part = 0;  // floats of a product's pieces
  const auto need = [&](const Tiling &t, uint64_t rows, uint64_t cols, bool sym) {
    if (t.parts == 1) return;
    const uint64_t ti = rows / t.tile, tj = cols / t.tile;
    const uint64_t n = (sym ? ti * (ti + 1) / 2 : ti * tj) * t.parts * t.tile * t.tile;
    part = n > part ? n : part;
  };
  need(p.gram, p.mp, p.mp, true);
  need(p.square, p.mp, p.mp, true);
  need(p.update, p.mp, p.np, false);
  return count * (kNormParts * 8 + 128 + 4 * part +
                  4 * (4 * uint64_t(p.mp) * p.np + (p.pairs ? 4 : 2) * uint64_t(p.mp) * p.mp));
}

template <class T, Mode M, bool MUON, int BM, int BN, int WM, int WN>
void launch_product(const Product &P, const MuonSet &S, uint32_t count) {
  constexpr int NW = (BM / WM) * (BN / WN);
  const uint32_t tiles = (M == Gram || M == Square ? P.ti * (P.ti + 1) / 2 : P.ti * P.tj) * count;
  product_kernel<T, M, MUON, BM, BN, WM, WN><<<tiles * P.parts, 64 * NW, 0, stream()>>>(P, S);
  if (P.parts > 1)
    join_kernel<T, M, MUON, BM, BN, WM, WN>
        <<<tiles * (BM / 32) * (BN / 32) / (kNsBlock / 64), kNsBlock, 0, stream()>>>(P, S);
}
template <class T, Mode M, bool MUON>
void product(const Plan &plan, const Tiling &how, Product &P, const MuonSet &S, uint32_t count) {
  P.parts = how.parts;
  P.ti = plan.mp / how.tile;
  P.tj = (M == Gram || M == Square ? plan.mp : plan.np) / how.tile;
  if (how.tile == 32) {
    const uint32_t tiles = (M == Gram || M == Square ? P.ti * (P.ti + 1) / 2 : P.ti * P.tj) * count;
    small_product_kernel<T, M, MUON><<<tiles, 64 * kSmallWaves, 0, stream()>>>(P, S);
  } else if (how.tile == 256) {
    launch_product<T, M, MUON, 256, 256, 128, 64>(P, S, count);
  } else if (how.tile == 128) {
    launch_product<T, M, MUON, 128, 128, 64, 64>(P, S, count);
  } else {
    launch_product<T, M, MUON, 64, 64, 32, 32>(P, S, count);
  }
}

// The iteration over `count` matrices: from G into O, or of a Muon set into its parameters.
template <class T, bool MUON>
void iterate(const Plan &plan, const Stack &G, const Stack &O, const MuonSet &S, uint32_t count,
             const NewtonSchulz &rule, void *work) {
  const uint64_t mn = 4 * uint64_t(plan.mp) * plan.np, mm = 4 * uint64_t(plan.mp) * plan.mp;
  double *norms = static_cast<double *>(work);
  float *xscale = reinterpret_cast<float *>(norms + uint64_t(count) * kNormParts);
  char *at = static_cast<char *>(work) + uint64_t(count) * (kNormParts * 8 + 128);
  const auto take = [&](uint64_t bytes, uint64_t pitch) {
    Lines l{at, pitch, bytes};
    at += count * bytes;
    return l;
  };
  Lines x = take(mn, 4 * uint64_t(plan.np)), y = take(mn, 4 * uint64_t(plan.np));
  Lines xt = take(mn, 4 * uint64_t(plan.mp)), yt = take(mn, 4 * uint64_t(plan.mp));
  const Lines a = take(mm, 4 * uint64_t(plan.mp)), s = take(mm, 4 * uint64_t(plan.mp));
  const Lines pa = plan.pairs ? take(mm, 4 * uint64_t(plan.mp)) : Lines{};
  const Lines s2 = plan.pairs ? take(mm, 4 * uint64_t(plan.mp)) : Lines{};
  float *partial = reinterpret_cast<float *>(at);

  const uint64_t size = uint64_t(G.rows) * G.cols;
  uint64_t parts = (size + 8 * kNsBlock - 1) / (8 * kNsBlock), most = 4096 / count + 1;
  parts = parts > most ? most : parts;
  const uint32_t np = uint32_t(parts > kNormParts ? kNormParts : parts);
  if constexpr (MUON) momentum_kernel<<<dim3(np, count), kNsBlock, 0, stream()>>>(S, size, norms);
  else norm_kernel<T><<<dim3(np, count), kNsBlock, 0, stream()>>>(G, MagicDiv::make(G.cols), norms);
  const bool tall = G.rows > G.cols;
  const dim3 grid((tall ? plan.mp : plan.np) / 64, (tall ? plan.np : plan.mp) / 64, count);
  start_kernel<T, MUON><<<grid, kNsBlock, 0, stream()>>>(G, S, norms, np, rule.eps, plan.growth, plan.room,
                                                       plan.scale.x, x, xt, xscale);
  const float sa = plan.scale.a, ss = plan.scale.s;
  Product P;
  memset(&P, 0, sizeof P);
  P.partial = partial;
  P.xscale = xscale;
  const auto gram = [&] {
    P.u = P.v = x, P.out = P.out_t = a, P.lines = plan.np / 32, P.alpha = sa;
    product<float, Gram, false>(plan, plan.gram, P, S, count);
  };
  // to = coef u v + beta in + gamma in2, of scales su, sv, so, si and s2
  const auto square = [&](const Lines &to, float so, float coef, const Lines &u, float su, const Lines &v, float sv,
                          float beta, const Lines &in, float si, float gamma = 0.0f, Lines in2 = Lines{}, float s2 = 1.0f) {
    P.u = u, P.v = v, P.in = P.in_t = in, P.in2 = in2, P.out = P.out_t = to;
    P.lines = plan.mp / 32;
    P.alpha = coef * (so / (su * sv)), P.beta = beta * (so / si), P.gamma = gamma * (so / s2);
    product<float, Square, false>(plan, plan.square, P, S, count);
  };
  for (int k = 0; k < rule.steps;) {
    const int steps = plan.pairs && k + 2 <= rule.steps ? 2 : 1;
    gram();
    square(s, ss, rule.c, a, sa, a, sa, rule.b, a, sa);
    Lines q = s;
    float identity = rule.a;
    if (steps == 2) {
      square(pa, sa, 1.0f, s, ss, a, sa, rule.a, a, sa);
      square(a, sa, 1.0f, s, ss, pa, sa, rule.a, pa, sa);
      square(s2, ss, rule.c, a, sa, a, sa, rule.b, a, sa);
      square(pa, ss, 1.0f, s2, ss, s, ss, rule.a, s, ss, rule.a, s2, ss);
      q = pa;
      identity *= rule.a;
    }
    k += steps;
    P.u = q, P.v = P.in_t = xt, P.in = x, P.out = y, P.out_t = yt, P.lines = plan.mp / 32;
    P.alpha = 1.0f / ss, P.beta = identity;
    if (k < rule.steps) {
      product<float, Update, false>(plan, plan.update, P, S, count);
      Lines z = x;
      x = y, y = z;
      z = xt, xt = yt, yt = z;
    } else {
      P.o = O;
      product<T, Final, MUON>(plan, plan.update, P, S, count);
    }
  }
  if (rule.steps == 0)
    copy_out_kernel<T, MUON><<<dim3(ceil_div(O.cols, kNsBlock), O.rows, count), kNsBlock, 0, stream()>>>(x, xt, xscale, O, S);
}

bool check_rule(const NewtonSchulz *r, const char *where) {
  if (!r) {
    report_error(where, "the rule is NULL");
    return false;
  }
  if (r->steps < 0 || r->steps > 1000 || !(r->eps >= 0.0f) || !std::isfinite(r->a) ||
      !std::isfinite(r->b) || !std::isfinite(r->c) || !std::isfinite(r->eps)) {
    report_error(where, "a rule needs 0 to 1000 steps, finite coefficients and eps of at least 0");
    return false;
  }
  const double most = range_of(*r).most;
  if (!(most <= 4.0)) {
    report_error(where, "the rule diverges: it takes singular values of 0 to 1 to %g", most);
    return false;
  }
  return true;
}

constexpr uint64_t kMaxExtent = 65535;             // of a matrix
constexpr uint64_t kNsBytes = uint64_t(8) << 30;  // workspace that stacks are cut to

// Matrices that go through the launches together.
uint64_t stack_share(uint64_t count, uint32_t rows, uint32_t cols) {
  const uint64_t mn = uint64_t(round_up(rows, 256)) * round_up(cols, 256);
  uint64_t c = kNsBytes / (16 * mn + 16 * mn);
  c = c < 1 ? 1 : c > 4096 ? 4096 : c;
  return count < c ? count : c;
}

bool matrix_stack(const Tensor *t, Stack &S, uint64_t &count, const char *name, const char *where) {
  if (!t || t->device != GPU || !is_float(t) || (t->ndim != 2 && t->ndim != 3)) {
    report_error(where, "%s must be a GPU matrix or stack of matrices of FLOAT32, FLOAT16 or BFLOAT16",
                 name);
    return false;
  }
  const uint64_t d = t->ndim - 2;
  count = d ? t->shape[0] : 1;
  if (t->shape[d] > kMaxExtent || t->shape[d + 1] > kMaxExtent) {
    report_error(where, "matrices of %llu x %llu are not supported", (unsigned long long)t->shape[d],
                 (unsigned long long)t->shape[d + 1]);
    return false;
  }
  if (numel(t) && !t->data) {
    report_error(where, "%s has no data", name);
    return false;
  }
  S.data = t->data;
  S.rows = uint32_t(t->shape[d]);
  S.cols = uint32_t(t->shape[d + 1]);
  S.sb = d ? int64_t(t->strides[0]) : 0;
  S.s0 = int64_t(t->strides[d]);
  S.s1 = int64_t(t->strides[d + 1]);
  return true;
}

// ------------------------------------------------------------------------- Muon

// Moment arrays that the library made (freed by plast_hip_muon_release).
std::mutex g_muon_mu;
std::unordered_set<Tensor **> g_muon_owned;

bool alloc_moments(Muon *o, Tensor **params, int count, const char *where) {
  Tensor **m = static_cast<Tensor **>(calloc(size_t(count), sizeof(Tensor *)));
  if (!m) {
    report_error(where, "host allocation of the moment array failed");
    return false;
  }
  for (int k = 0; k < count; ++k) {
    const Tensor *p = params[k];
    if (!p) continue;
    Tensor *t = static_cast<Tensor *>(calloc(1, sizeof(Tensor)));
    const uint64_t n = numel(p);
    if (!t || (n && hipMalloc(&t->data, n * sizeof(float)) != hipSuccess)) {
      free(t);
      report_error(where, "allocation of a moment tensor (%llu floats) failed", (unsigned long long)n);
      continue;
    }
    t->ndim = p->ndim;
    uint64_t s = 1;
    for (uint64_t d = p->ndim; d-- > 0;) {
      t->shape[d] = p->shape[d];
      t->strides[d] = s;
      s *= p->shape[d];
    }
    t->dtype = FLOAT32;
    t->device = GPU;
    if (n) zeros_hip(t, n);
    m[k] = t;
  }
  o->m = m;
  std::lock_guard<std::mutex> lk(g_muon_mu);
  g_muon_owned.insert(m);
  return true;
}

bool f32_matrix(const Tensor *t, const Tensor *shape_of) {
  return t && t->device == GPU && t->dtype == FLOAT32 && t->ndim == 2 && contiguous(t) && (t->data || numel(t) == 0) &&
         same_shape(t, shape_of);
}

}  // namespace
}  // namespace plast

using namespace plast;

extern "C" {

void newton_schulz_hip(const Tensor *g, Tensor *out, const NewtonSchulz *rule) {
  const char *where = "newton_schulz_hip";
  Stack G, O;
  uint64_t count = 0, same = 0;
  if (!check_rule(rule, where) || !matrix_stack(g, G, count, "g", where) ||
      !matrix_stack(out, O, same, "out", where))
    return;
  if (g->dtype != out->dtype || !same_shape(g, out)) {
    report_error(where, "out must have g's type and shape");
    return;
  }
  if (overlapping(out)) {
    report_error(where, "elements of out overlap");
    return;
  }
  if (numel(g) == 0 || !ensure_init()) return;
  const uint64_t share = stack_share(count, G.rows, G.cols), item = float_bytes(g);
  const Plan plan = make_plan(G.rows, G.cols, share, *rule);
  void *work = workspace(ns_bytes(plan, share));
  if (!work) return;
  MuonSet none;
  memset(&none, 0, sizeof none);
  for (uint64_t b = 0; b < count; b += share) {
    Stack Gb = G, Ob = O;
    Gb.data = static_cast<const char *>(G.data) + int64_t(b) * G.sb * int64_t(item);
    Ob.data = static_cast<const char *>(O.data) + int64_t(b) * O.sb * int64_t(item);
    with_float_type(g->dtype, [&](auto t) {
      typedef decltype(t) T;
      iterate<T, false>(plan, Gb, Ob, none, uint32_t(count - b < share ? count - b : share), *rule, work);
    });
  }
  finish(where);
}

void muon_step_hip(Muon *optimizer, Tensor **parameters, int num_parameters) {
  const char *where = "muon_step_hip";
  if (!optimizer) {
    report_error(where, "optimizer is NULL");
    return;
  }
  if (!check_rule(&optimizer->rule, where)) return;
  if (num_parameters <= 0 || !parameters) return;
  // everything is checked before anything is written
  for (int k = 0; k < num_parameters; ++k) {
    const Tensor *p = parameters[k];
    if (!p || !p->grad) continue;
    if (!f32_matrix(p, p) || !f32_matrix(p->grad, p) || p->shape[0] > kMaxExtent || p->shape[1] > kMaxExtent) {
      report_error(where, "parameter %d is not a contiguous FLOAT32 matrix with such a gradient, or too "
                   "large", k);
      return;
    }
  }
  if (!ensure_init()) return;
  if (!optimizer->m && capturing()) {  // a replay would zero them each time
    report_error(where, "the first step makes the moments: run one before capturing");
    return;
  }
  if (!optimizer->m && !alloc_moments(optimizer, parameters, num_parameters, where)) return;
  for (int k = 0; k < num_parameters; ++k)
    if (parameters[k] && parameters[k]->grad && !f32_matrix(optimizer->m[k], parameters[k])) {
      report_error(where, "moment tensor of parameter %d is missing or not a contiguous FLOAT32 matrix "
                   "of its shape", k);
      return;
    }
  // the parameters of each shape, and a workspace for the largest, before anything is written
  struct Group {
    std::vector<int> which;
    uint64_t share;
    Plan plan;
  };
  std::vector<char> done(size_t(num_parameters), 0);
  std::vector<Group> groups;
  uint64_t bytes = 0;
  for (int k = 0; k < num_parameters; ++k) {
    const Tensor *first = parameters[k];
    if (done[k] || !first || !first->grad || numel(first) == 0) continue;
    Group g;
    for (int j = k; j < num_parameters; ++j)
      if (!done[j] && parameters[j] && parameters[j]->grad && same_shape(parameters[j], first)) {
        g.which.push_back(j);
        done[j] = 1;
      }
    const uint32_t rows = uint32_t(first->shape[0]), cols = uint32_t(first->shape[1]);
    g.share = stack_share(g.which.size(), rows, cols);
    if (g.share > kPointers) g.share = kPointers;
    g.plan = make_plan(rows, cols, g.share, optimizer->rule);
    const uint64_t need = ns_bytes(g.plan, g.share);
    bytes = need > bytes ? need : bytes;
    groups.push_back(std::move(g));
  }
  if (groups.empty()) return;
  void *work = workspace(bytes);
  if (!work) return;
  for (const Group &group : groups) {
    const Tensor *first = parameters[group.which[0]];
    const uint32_t rows = uint32_t(first->shape[0]), cols = uint32_t(first->shape[1]);
    MuonSet S;
    memset(&S, 0, sizeof S);
    S.rule.momentum = optimizer->momentum;
    S.rule.nesterov = optimizer->nesterov;
    S.rule.keep = 1.0f - optimizer->lr * optimizer->weight_decay;
    S.rule.scale = optimizer->lr * sqrtf(rows > cols ? float(rows) / float(cols) : 1.0f);
    const Stack shape{nullptr, rows, cols, 0, int64_t(cols), 1};
    for (size_t b = 0; b < group.which.size(); b += group.share) {
      const size_t c = group.which.size() - b < group.share ? group.which.size() - b : group.share;
      for (size_t j = 0; j < c; ++j) {
        const int at = group.which[b + j];
        S.p[j] = static_cast<float *>(parameters[at]->data);
        S.g[j] = static_cast<const float *>(parameters[at]->grad->data);
        S.m[j] = static_cast<float *>(optimizer->m[at]->data);
      }
      iterate<float, true>(group.plan, shape, shape, S, uint32_t(c), optimizer->rule, work);
    }
  }
  finish(where);
}

void plast_hip_muon_release(Muon *optimizer, int num_parameters) {
  if (!optimizer || !optimizer->m) return;
  std::lock_guard<std::mutex> lk(g_muon_mu);
  if (!g_muon_owned.count(optimizer->m)) return;
  for (int k = 0; k < num_parameters; ++k) {
    Tensor *t = optimizer->m[k];
    if (!t) continue;
    if (t->data) (void)hipFree(t->data);
    free(t);
  }
  g_muon_owned.erase(optimizer->m);
  free(optimizer->m);
  optimizer->m = nullptr;
}

}  // extern "C"
