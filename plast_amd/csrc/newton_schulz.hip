// newton_schulz.hip — the Newton-Schulz orthogonalisation of a matrix, or of each of a stack, and the
// Muon optimizer step built on it.
//
// With G on the side with m <= n rows (transposed where it has more rows than columns) and
// X = G / (|G| + eps), Frobenius norm, each of `steps` iterations is
//   A = X X^T (m x m),  S = b A + c A A (m x m),  X = a X + S X (m x n).
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
constexpr uint32_t kNormParts = 64;  // workgroups that share a matrix's norm

// A stack of matrices with any strides, in elements.
struct Stack {
  const void *data;
  uint32_t rows, cols;
  int64_t sb, s0, s1;
};

// |G|^2 in 64 bits, where neither the squares nor their sum overflow or vanish: one partial sum
// per workgroup, then one per matrix in norm_scale.
template <class T>
__global__ __launch_bounds__(kNsBlock) void norm_kernel(Stack G, double *part) {
  __shared__ double lds[kNsBlock / 64];
  const T *g = static_cast<const T *>(G.data) + int64_t(blockIdx.y) * G.sb;
  double s = 0.0;
  for (uint32_t i = blockIdx.x; i < G.rows; i += gridDim.x)
    for (uint32_t j = threadIdx.x; j < G.cols; j += kNsBlock) {
      const double v = double(float(g[int64_t(i) * G.s0 + int64_t(j) * G.s1]));
      s += v * v;
    }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < kNsBlock / 64; ++k) s += lds[k];
    part[uint64_t(blockIdx.y) * kNormParts + blockIdx.x] = s;
  }
}

// 1 / (|G| + eps) of matrix b from its partial sums, by every thread.
__device__ __forceinline__ double norm_scale(const double *part, uint32_t b, uint32_t parts, float eps) {
  double s = 0.0;
  for (uint32_t k = 0; k < parts; ++k) s += part[uint64_t(b) * kNormParts + k];
  return 1.0 / (sqrt(s) + double(eps));
}

// X[b] [m, n] = G[b] * scale, transposed where G has more rows than columns.
template <class T>
__global__ __launch_bounds__(kNsBlock) void start_kernel(Stack G, const double *part, uint32_t parts,
                                                         float eps, float *X, uint32_t m, uint32_t n) {
  const uint32_t b = blockIdx.z, i = blockIdx.y, j = blockIdx.x * kNsBlock + threadIdx.x;
  if (j >= n) return;
  const double scale = norm_scale(part, b, parts, eps);
  const bool tall = G.rows > G.cols;
  const T *g = static_cast<const T *>(G.data) + int64_t(b) * G.sb;
  const float v = float(g[int64_t(tall ? j : i) * G.s0 + int64_t(tall ? i : j) * G.s1]);
  X[(uint64_t(b) * m + i) * n + j] = float(double(v) * scale);
}

template <class T>
__global__ __launch_bounds__(kNsBlock) void finish_kernel(const float *X, uint32_t m, uint32_t n, Stack O) {
  const uint32_t b = blockIdx.z, i = blockIdx.y, j = blockIdx.x * kNsBlock + threadIdx.x;
  if (j >= n) return;
  const bool tall = O.rows > O.cols;
  T *o = static_cast<T *>(const_cast<void *>(O.data)) + int64_t(b) * O.sb;
  o[int64_t(tall ? j : i) * O.s0 + int64_t(tall ? i : j) * O.s1] = T(X[(uint64_t(b) * m + i) * n + j]);
}

// C = alpha A B + beta D over row-major C, D [p, q]; A[i, k] and B[k, j] by strides. 64x64 tiles,
// 4x4 outputs a lane, both operands staged through LDS.
struct Product {
  const float *a, *b, *d;
  float *c;
  uint32_t p, q, k;
  int64_t a0, a1, b0, b1;      // strides
  uint64_t ab, bb, cb;         // from one matrix of the stack to the next
  float alpha, beta;
};
__global__ __launch_bounds__(kNsBlock) void product_kernel(Product P) {
  __shared__ float la[16][64 + 4], lb[16][64 + 4];
  const uint32_t i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
  const float *a = P.a + blockIdx.z * P.ab, *b = P.b + blockIdx.z * P.bb;
  const int ti = threadIdx.x / 16, tj = threadIdx.x % 16;
  float acc[4][4] = {};
  for (uint32_t k0 = 0; k0 < P.k; k0 += 16) {
    for (int e = threadIdx.x; e < 16 * 64; e += kNsBlock) {
      const uint32_t kk = e % 16, r = e / 16;
      la[kk][r] = i0 + r < P.p && k0 + kk < P.k ? a[int64_t(i0 + r) * P.a0 + int64_t(k0 + kk) * P.a1] : 0.0f;
      lb[kk][r] = j0 + r < P.q && k0 + kk < P.k ? b[int64_t(k0 + kk) * P.b0 + int64_t(j0 + r) * P.b1] : 0.0f;
    }
    __syncthreads();
    for (int kk = 0; kk < 16; ++kk)
      for (int u = 0; u < 4; ++u)
        for (int v = 0; v < 4; ++v)
          acc[u][v] = __builtin_fmaf(la[kk][ti * 4 + u], lb[kk][tj * 4 + v], acc[u][v]);
    __syncthreads();
  }
  for (int u = 0; u < 4; ++u)
    for (int v = 0; v < 4; ++v) {
      const uint32_t i = i0 + ti * 4 + u, j = j0 + tj * 4 + v;
      if (i >= P.p || j >= P.q) continue;
      const uint64_t at = blockIdx.z * P.cb + uint64_t(i) * P.q + j;
      P.c[at] = P.alpha * acc[u][v] + (P.d ? P.beta * P.d[at] : 0.0f);
    }
}

void product(const Product &P, uint32_t count) {
  product_kernel<<<dim3(ceil_div(P.q, 64), ceil_div(P.p, 64), count), kNsBlock, 0, stream()>>>(P);
}

// The iteration over `count` matrices G into O, in a workspace of ns_bytes(count, m, n) bytes.
uint64_t ns_bytes(uint64_t count, uint64_t m, uint64_t n) {
  return count * (kNormParts * sizeof(double) + (2 * m * n + 2 * m * m) * sizeof(float));
}
void iterate(const Stack &G, DTYPE type, const Stack &O, uint32_t count, const NewtonSchulz &rule,
             void *work) {
  const uint32_t m = G.rows < G.cols ? G.rows : G.cols, n = G.rows < G.cols ? G.cols : G.rows;
  const uint64_t mn = uint64_t(m) * n, mm = uint64_t(m) * m;
  double *part = static_cast<double *>(work);
  float *x = reinterpret_cast<float *>(part + uint64_t(count) * kNormParts), *y = x + count * mn;
  float *a = y + count * mn, *s = a + count * mm;
  const uint32_t parts = G.rows < kNormParts ? G.rows : kNormParts;
  const dim3 grid(ceil_div(n, kNsBlock), m, count);
  with_float_type(type, [&](auto t) {
    norm_kernel<decltype(t)><<<dim3(parts, count), kNsBlock, 0, stream()>>>(G, part);
    start_kernel<decltype(t)><<<grid, kNsBlock, 0, stream()>>>(G, part, parts, rule.eps, x, m, n);
  });
  for (int k = 0; k < rule.steps; ++k) {
    product(Product{x, x, nullptr, a, m, m, n, n, 1, 1, n, mn, mn, mm, 1.0f, 0.0f}, count);
    product(Product{a, a, a, s, m, m, m, m, 1, m, 1, mm, mm, mm, rule.c, rule.b}, count);
    product(Product{s, x, x, y, m, n, m, m, 1, n, 1, mm, mn, mn, 1.0f, rule.a}, count);
    float *z = x;
    x = y, y = z;
  }
  with_float_type(type, [&](auto t) {
    finish_kernel<decltype(t)><<<grid, kNsBlock, 0, stream()>>>(x, m, n, O);
  });
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
  return true;
}

constexpr uint64_t kMaxExtent = 65535;             // of a matrix
constexpr uint64_t kNsBytes = uint64_t(8) << 30;  // workspace that stacks are cut to

// Matrices that go through the launches together.
uint64_t stack_share(uint64_t count, uint64_t bytes_each) {
  uint64_t c = kNsBytes / bytes_each;
  c = c < 1 ? 1 : c > 65535 ? 65535 : c;
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

// Whether two elements of t can lie at one address: an axis of several elements, in order of their
// strides, steps no further than what the ones below it span.
bool overlapping(const Tensor *t) {
  uint64_t need = 1;
  bool done[PLAST_MAX_NDIM] = {};
  for (uint64_t k = 0; k < t->ndim; ++k) {
    uint64_t at = t->ndim;
    for (uint64_t d = 0; d < t->ndim; ++d)
      if (!done[d] && (at == t->ndim || t->strides[d] < t->strides[at])) at = d;
    done[at] = true;
    if (t->shape[at] <= 1) continue;
    if (t->strides[at] < need) return true;
    need = t->strides[at] * t->shape[at];
  }
  return false;
}

// ------------------------------------------------------------------------- Muon

struct MuonRule {
  float momentum, keep, scale;  // keep: 1 - lr decay; scale: lr sqrt(max(1, rows / cols))
  int nesterov;
};

__global__ __launch_bounds__(kNsBlock) void momentum_kernel(const float *g, float *m, float *u, uint64_t n,
                                                            MuonRule R) {
  for (uint64_t i = uint64_t(blockIdx.x) * kNsBlock + threadIdx.x; i < n; i += uint64_t(gridDim.x) * kNsBlock) {
    const float gi = g[i];
    const float v = R.momentum * m[i] + (1.0f - R.momentum) * gi;
    m[i] = v;
    u[i] = R.nesterov ? (1.0f - R.momentum) * gi + R.momentum * v : v;
  }
}

__global__ __launch_bounds__(kNsBlock) void apply_kernel(float *p, const float *o, uint64_t n, MuonRule R) {
  for (uint64_t i = uint64_t(blockIdx.x) * kNsBlock + threadIdx.x; i < n; i += uint64_t(gridDim.x) * kNsBlock)
    p[i] = p[i] * R.keep - R.scale * o[i];
}

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
  const uint64_t m = G.rows < G.cols ? G.rows : G.cols, n = G.rows < G.cols ? G.cols : G.rows;
  const uint64_t share = stack_share(count, ns_bytes(1, m, n)), item = float_bytes(g);
  void *work = workspace(ns_bytes(share, m, n));
  if (!work) return;
  for (uint64_t b = 0; b < count; b += share) {
    Stack Gb = G, Ob = O;
    Gb.data = static_cast<const char *>(G.data) + int64_t(b) * G.sb * int64_t(item);
    Ob.data = static_cast<const char *>(O.data) + int64_t(b) * O.sb * int64_t(item);
    iterate(Gb, g->dtype, Ob, uint32_t(count - b < share ? count - b : share), *rule, work);
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
  if (!optimizer->m && !alloc_moments(optimizer, parameters, num_parameters, where)) return;
  for (int k = 0; k < num_parameters; ++k)
    if (parameters[k] && parameters[k]->grad && !f32_matrix(optimizer->m[k], parameters[k])) {
      report_error(where, "moment tensor of parameter %d is missing or not a contiguous FLOAT32 matrix "
                   "of its shape", k);
      return;
    }
  std::vector<char> done(size_t(num_parameters), 0);
  for (int k = 0; k < num_parameters; ++k) {
    const Tensor *first = parameters[k];
    if (done[k] || !first || !first->grad || numel(first) == 0) continue;
    std::vector<int> same;  // the parameters of this shape
    for (int j = k; j < num_parameters; ++j)
      if (!done[j] && parameters[j] && parameters[j]->grad && same_shape(parameters[j], first)) {
        same.push_back(j);
        done[j] = 1;
      }
    const uint64_t rows = first->shape[0], cols = first->shape[1], size = rows * cols;
    const uint64_t m = rows < cols ? rows : cols, n = rows < cols ? cols : rows;
    const uint64_t each = ns_bytes(1, m, n) + size * sizeof(float);
    const uint64_t share = stack_share(same.size(), each);
    char *work = static_cast<char *>(workspace(share * each));
    if (!work) return;
    float *u = reinterpret_cast<float *>(work + ns_bytes(share, m, n));
    MuonRule R;
    R.momentum = optimizer->momentum;
    R.nesterov = optimizer->nesterov;
    R.keep = 1.0f - optimizer->lr * optimizer->weight_decay;
    R.scale = optimizer->lr * sqrtf(rows > cols ? float(rows) / float(cols) : 1.0f);
    const Stack U{u, uint32_t(rows), uint32_t(cols), int64_t(size), int64_t(cols), 1};
    const unsigned grid = unsigned(size < (uint64_t(1) << 20) ? ceil_div(size, kNsBlock) : 4096);
    for (size_t b = 0; b < same.size(); b += share) {
      const size_t c = same.size() - b < share ? same.size() - b : share;
      for (size_t j = 0; j < c; ++j) {
        const Tensor *p = parameters[same[b + j]];
        momentum_kernel<<<grid, kNsBlock, 0, stream()>>>(
            static_cast<const float *>(p->grad->data), static_cast<float *>(optimizer->m[same[b + j]]->data),
            u + j * size, size, R);
      }
      iterate(U, FLOAT32, U, uint32_t(c), optimizer->rule, work);
      for (size_t j = 0; j < c; ++j)
        apply_kernel<<<grid, kNsBlock, 0, stream()>>>(static_cast<float *>(parameters[same[b + j]]->data),
                                                      u + j * size, size, R);
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
