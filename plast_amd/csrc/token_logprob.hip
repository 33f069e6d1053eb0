// token_logprob.hip — log-probabilities of given tokens with the rows' entropies, their most likely
// alternatives, and the gradient; the distribution of a row is p = softmax(x / T).
//
// The mathematics is in base 2, the hardware's exponential. With c = log2(e) / T, m the row's largest
// logit and z_j = c x_j - c m:
//   s = sum_j 2^z_j,  w = sum_j 2^z_j z_j,
//   log p_j = (x_j - m) / T - ln2 log2 s,  H = -sum_j p_j log p_j = ln2 (log2 s - w / s).
// c m is rounded once and z_j = fma(c, x_j, -c m) once more: the first rounding, r = c m - round(c m),
// moves every z_j alike, so p and H do not see it, and log p takes it out of log2 s again; the second is
// relative to z_j itself, however large the logits are.
// Gradient for upstream u of log p[token] and h of H:
//   dx_j = (u ([j = token] - p_j) - h p_j (log p_j + H)) / T
//        = u / T [j = token] - 2^z_j (A + B z_j),
//   B = h ln2 / (T s),  A = (u + h H) / (T s) - B log2 s.
#include <cfloat>
#include <cmath>

#include "half_types.hpp"

namespace plast {
namespace {

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kInf = __builtin_huge_valf();
constexpr int kRowBlock = 256;  // lanes of a workgroup

// Where row `r` of the leading axes starts, in elements, in x and in its gradient.
struct RowMap {
  int rank;
  MagicDiv ext[kMaxRank];
  int64_t x[kMaxRank], g[kMaxRank];
};
struct RowAt {
  int64_t x, g;
};
__device__ __forceinline__ RowAt row_at(const RowMap &M, uint32_t r) {
  RowAt at{0, 0};
  for (int d = M.rank - 1; d > 0; --d) {
    const uint32_t q = M.ext[d].div(r), i = r - q * M.ext[d].d;
    at.x += int64_t(i) * M.x[d];
    at.g += int64_t(i) * M.g[d];
    r = q;
  }
  at.x += int64_t(r) * M.x[0];
  at.g += int64_t(r) * M.g[0];
  return at;
}

// What a launch needs of its tensors.
struct TokenArgs {
  const void *x;
  void *dx;
  const int32_t *tokens;
  float *stats, *entropy, *logp;
  const float *dlogp, *dentropy;  // either may be null: zero
  float *top_logp;
  int32_t *top_ids;
  uint32_t top;
  uint32_t rows, vocab;
  float c;      // log2(e) / T
  float inv_t;  // 1 / T
  RowMap map;
};

// The exponent z of a logit. Where c m overflows, c (x - m) is taken instead.
struct RowRef {
  float c, m, cm;
  bool far;
  __device__ __forceinline__ RowRef(float c_, float m_) : c(c_), m(m_), cm(c_ * m_) {
    far = !(fabsf(cm) < 1e38f);
  }
  __device__ __forceinline__ float z(float x) const {
    return far ? (x - m) * c : __builtin_fmaf(x, c, -cm);
  }
  // What the rounding of c m adds to every z.
  __device__ __forceinline__ float shift() const { return far ? 0.0f : __builtin_fmaf(c, m, -cm); }
};

// Adds a logit's terms to s and w; a masked logit (z = -inf) adds nothing.
__device__ __forceinline__ void add_terms(float z, float &s, float &w) {
  const float e = __builtin_amdgcn_exp2f(z);
  s += e;
  w = __builtin_fmaf(e, fmaxf(z, -FLT_MAX), w);
}

template <int W>
__device__ __forceinline__ float block_reduce(float v, float *lds, bool maximum) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const float o = __shfl_xor(v, m);
    v = maximum ? fmaxf(v, o) : v + o;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float r = lds[0];
#pragma unroll
  for (int k = 1; k < W; ++k) r = maximum ? fmaxf(r, lds[k]) : r + lds[k];
  return r;
}

// A logit's place in the order of alternatives: larger first, equal logits (both zeros too) by the
// lower index, NaN above all. No key is 0.
__device__ __forceinline__ uint64_t order_key(float v, uint32_t j) {
  v += 0.0f;  // -0 counts as +0
  const uint32_t b = __float_as_uint(v);
  const uint32_t k = v != v ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
  return uint64_t(k) << 32 | (0xffffffffu - j);
}

// log p of a logit from the row's statistics.
__device__ __forceinline__ float log_p(const TokenArgs &A, float x, float m, float l0) {
  return m == -kInf ? -kInf : (x - m) * A.inv_t - kLn2 * l0;
}

// The row's results, by one lane. s and w are over the whole row.
__device__ __forceinline__ void row_out(const TokenArgs &A, uint32_t row, int32_t token, float x_token,
                                        float m, float s, float w) {
  if (m == -kInf) {  // no logit that is not -inf
    A.logp[row] = uint32_t(token) < A.vocab ? -kInf : __builtin_nanf("");
    A.entropy[row] = 0.0f;
    A.stats[2 * row] = -kInf;
    A.stats[2 * row + 1] = 0.0f;
    return;
  }
  const float l = log2f(s);
  const RowRef ref(A.c, m);
  const float h = kLn2 * (l - w / s);
  const float l0 = l - ref.shift();
  A.logp[row] = uint32_t(token) < A.vocab ? log_p(A, x_token, m, l0) : __builtin_nanf("");
  A.entropy[row] = h < 0.0f ? 0.0f : h;
  A.stats[2 * row] = m;
  A.stats[2 * row + 1] = l0;
}

__device__ __forceinline__ void pad_out(const TokenArgs &A, uint32_t row) {
  A.logp[row] = 0.0f;
  A.entropy[row] = 0.0f;
  A.stats[2 * row] = -kInf;
  A.stats[2 * row + 1] = 0.0f;
}

// One workgroup per row: the maximum, then the sums, then an argmax per alternative.
template <class T>
__global__ __launch_bounds__(kRowBlock) void fwd_kernel(TokenArgs A) {
  __shared__ float lds[4];
  __shared__ uint64_t keys[4];
  const uint32_t row = blockIdx.x, V = A.vocab;
  const int32_t token = A.tokens[row];
  const uint32_t top = A.top;
  if (token < 0) {
    if (threadIdx.x == 0) pad_out(A, row);
    if (threadIdx.x < top) {
      A.top_logp[uint64_t(row) * top + threadIdx.x] = -kInf;
      A.top_ids[uint64_t(row) * top + threadIdx.x] = -1;
    }
    return;
  }
  const T *x = static_cast<const T *>(A.x) + row_at(A.map, row).x;
  float m = -kInf;
  for (uint32_t j = threadIdx.x; j < V; j += kRowBlock) m = fmaxf(m, float(x[j]));
  m = block_reduce<4>(m, lds, true);
  const RowRef ref(A.c, m);
  float s = 0.0f, w = 0.0f;
  bool nan = false;
  for (uint32_t j = threadIdx.x; j < V; j += kRowBlock) {
    const float v = float(x[j]);
    nan = nan || v != v;
    if (m != -kInf) add_terms(ref.z(v), s, w);
  }
  if (nan) s = __builtin_nanf("");
  s = block_reduce<4>(s, lds, false);
  w = block_reduce<4>(w, lds, false);
  if (s != s) m = s;  // a NaN or an infinite logit
  if (threadIdx.x == 0)
    row_out(A, row, token, uint32_t(token) < V ? float(x[token]) : 0.0f, m, s, w);
  uint64_t last = ~uint64_t(0);
  for (uint32_t k = 0; k < top; ++k) {
    uint64_t best = 0;
    for (uint32_t j = threadIdx.x; j < V; j += kRowBlock) {
      const uint64_t key = order_key(float(x[j]), j);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      const uint64_t o = __shfl_xor((unsigned long long)best, d);
      best = o > best ? o : best;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) keys[threadIdx.x >> 6] = best;
    __syncthreads();
    for (int d = 0; d < 4; ++d) best = keys[d] > best ? keys[d] : best;
    if (threadIdx.x == 0) {
      const uint64_t at = uint64_t(row) * top + k;
      const uint32_t j = 0xffffffffu - uint32_t(best);
      A.top_ids[at] = best ? int32_t(j) : -1;
      A.top_logp[at] = best ? log_p(A, float(x[j]), m, log2f(s) - ref.shift()) : -kInf;
    }
    last = best;
  }
}

// One workgroup per row.
template <class T, bool ADD>
__global__ __launch_bounds__(kRowBlock) void bwd_kernel(TokenArgs A) {
  const uint32_t row = blockIdx.x, V = A.vocab;
  const int32_t token = A.tokens[row];
  const RowAt at = row_at(A.map, row);
  T *dx = static_cast<T *>(A.dx) + at.g;
  const float m = A.stats[2 * row];
  const RowRef ref(A.c, m);
  const float l = A.stats[2 * row + 1] + ref.shift();
  if (token < 0 || m == -kInf) {
    if (!ADD)
      for (uint32_t j = threadIdx.x; j < V; j += kRowBlock) dx[j] = T(0.0f);
    return;
  }
  const T *x = static_cast<const T *>(A.x) + at.x;
  const float u = A.dlogp ? A.dlogp[row] : 0.0f, h = A.dentropy ? A.dentropy[row] : 0.0f;
  const float r = A.inv_t * __builtin_amdgcn_exp2f(-l);  // 1 / (T s)
  const float b = h * kLn2 * r;
  float a = (u + h * A.entropy[row]) * r - b * l;
  if (uint32_t(token) >= V) a = __builtin_nanf("");
  for (uint32_t j = threadIdx.x; j < V; j += kRowBlock) {
    const float z = fmaxf(ref.z(float(x[j])), -300.0f);  // 2^-300 = 0; masked logits stay finite
    float d = -__builtin_amdgcn_exp2f(z) * __builtin_fmaf(b, z, a);
    if (j == uint32_t(token)) d += u * A.inv_t;
    if (ADD) d += float(dx[j]);
    dx[j] = T(d);
  }
}

// ------------------------------------------------------------------------- host

bool f32_vector(const Tensor *t, uint64_t n) {
  return t && t->device == GPU && t->dtype == FLOAT32 && numel(t) == n && contiguous(t) && (t->data || n == 0);
}

// Checks x, the tokens and the temperature; fills the row map (of x and, where given, its gradient).
bool token_args(TokenArgs &A, const Tensor *x, const Tensor *dx, const Tensor *tokens, float temp,
                const char *where) {
  memset(&A, 0, sizeof A);
  if (!x || !tokens) {
    report_error(where, "an input is NULL");
    return false;
  }
  if (x->device != GPU || !is_float(x) || x->ndim < 1 || x->ndim > PLAST_MAX_NDIM) {
    report_error(where, "x must be a GPU tensor of FLOAT32, FLOAT16 or BFLOAT16 with a last axis");
    return false;
  }
  const uint64_t V = x->shape[x->ndim - 1], n = numel(x);
  if (V < 1 || V >= uint64_t(1) << 31) {
    report_error(where, "rows of %llu logits are not supported", (unsigned long long)V);
    return false;
  }
  const uint64_t N = n / V;
  if (N >= uint64_t(1) << 31) {
    report_error(where, "%llu rows are not supported", (unsigned long long)N);
    return false;
  }
  if (V > 1 && x->strides[x->ndim - 1] != 1) {
    report_error(where, "the last axis of x must be contiguous, not strided by %llu",
                 (unsigned long long)x->strides[x->ndim - 1]);
    return false;
  }
  if (tokens->device != GPU || tokens->dtype != INT32 || numel(tokens) != N || !contiguous(tokens)) {
    report_error(where, "tokens must be a contiguous INT32 GPU tensor of %llu elements",
                 (unsigned long long)N);
    return false;
  }
  if (!(temp > 0.0f && temp <= FLT_MAX)) {
    report_error(where, "the temperature must be finite and above 0, not %g", double(temp));
    return false;
  }
  if (n && (!x->data || !tokens->data)) {
    report_error(where, "an input has no data");
    return false;
  }
  Space s;
  s.rank = int(x->ndim) - 1;
  s.nops = 2;
  for (int d = 0; d < s.rank; ++d) {
    s.shape[d] = x->shape[d];
    s.st[0][d] = int64_t(x->strides[d]);
    s.st[1][d] = dx ? int64_t(dx->strides[d]) : 0;
  }
  if (dx) {
    if (dx->device != GPU || dx->dtype != x->dtype || !same_shape(x, dx) || (n && !dx->data) ||
        (V > 1 && dx->strides[x->ndim - 1] != 1)) {
      report_error(where, "the gradient of x must have x's type and shape and a contiguous last axis");
      return false;
    }
    for (int d = 0; d < s.rank; ++d)
      if (x->shape[d] > 1 && dx->strides[d] < V) {
        report_error(where, "rows of x's gradient overlap along axis %d", d);
        return false;
      }
  }
  if (n) collapse(s);
  A.x = x->data;
  A.dx = dx ? dx->data : nullptr;
  A.tokens = static_cast<const int32_t *>(tokens->data);
  A.rows = uint32_t(N);
  A.vocab = uint32_t(V);
  A.inv_t = 1.0f / temp;
  A.c = float(double(1.4426950408889634074) / double(temp));
  if (!(A.c <= FLT_MAX)) {
    report_error(where, "the temperature %g is too small", double(temp));
    return false;
  }
  A.map.rank = s.rank;
  for (int d = 0; n && d < s.rank; ++d) {
    A.map.ext[d] = MagicDiv::make(uint32_t(s.shape[d]));
    A.map.x[d] = s.st[0][d];
    A.map.g[d] = s.st[1][d];
  }
  return true;
}

void launch_forward(const TokenArgs &A, DTYPE type) {
  with_float_type(type, [&](auto t) {
    fwd_kernel<decltype(t)><<<A.rows, kRowBlock, 0, stream()>>>(A);
  });
}

void launch_backward(const TokenArgs &A, DTYPE type, bool add) {
  with_float_type(type, [&](auto t) {
    if (add) bwd_kernel<decltype(t), true><<<A.rows, kRowBlock, 0, stream()>>>(A);
    else bwd_kernel<decltype(t), false><<<A.rows, kRowBlock, 0, stream()>>>(A);
  });
}

// The float vectors of a call.
bool token_vectors(TokenArgs &A, const Tensor *stats, const Tensor *entropy, const Tensor *logp,
                   const char *where) {
  const uint64_t N = A.rows;
  if (!f32_vector(stats, 2 * N) || !f32_vector(entropy, N) || !f32_vector(logp, N)) {
    report_error(where, "stats, entropy and logp must be contiguous FLOAT32 GPU tensors of 2 N, N and "
                 "N elements, N = %llu", (unsigned long long)N);
    return false;
  }
  A.stats = static_cast<float *>(stats->data);
  A.entropy = static_cast<float *>(entropy->data);
  A.logp = static_cast<float *>(logp->data);
  return true;
}

// An upstream gradient: none counts as zero.
bool upstream(const Tensor *g, uint64_t n, const float **out, const char *where) {
  *out = nullptr;
  if (!g) return true;
  if (!f32_vector(g, n)) {
    report_error(where, "an upstream gradient must be a contiguous FLOAT32 GPU tensor of %llu elements",
                 (unsigned long long)n);
    return false;
  }
  *out = static_cast<const float *>(g->data);
  return true;
}

}  // namespace
}  // namespace plast

using namespace plast;

extern "C" {

void token_logprob_hip_forward(const Tensor **inputs, Tensor *output, KernelParams params) {
  const char *where = "token_logprob_hip_forward";
  TokenArgs A;
  if (!token_args(A, inputs[0], nullptr, inputs[1], params.fval, where) ||
      !token_vectors(A, inputs[2], inputs[3], output, where))
    return;
  if (params.dim > PLAST_TOP_MAX) {
    report_error(where, "%llu alternatives are more than %d", (unsigned long long)params.dim,
                 PLAST_TOP_MAX);
    return;
  }
  A.top = uint32_t(params.dim);
  if (A.top) {
    const uint64_t n = uint64_t(A.rows) * A.top;
    const Tensor *ids = inputs[5];
    if (!f32_vector(inputs[4], n) || !ids || ids->device != GPU || ids->dtype != INT32 ||
        numel(ids) != n || !contiguous(ids) || (n && !ids->data)) {
      report_error(where, "top_logp and top_ids must be contiguous FLOAT32 and INT32 GPU tensors of "
                   "%llu elements", (unsigned long long)n);
      return;
    }
    A.top_logp = static_cast<float *>(inputs[4]->data);
    A.top_ids = static_cast<int32_t *>(ids->data);
  }
  if (A.rows == 0 || !ensure_init()) return;
  launch_forward(A, inputs[0]->dtype);
  finish(where);
}

void token_logprob_hip_backward(Tensor **inputs, const Tensor *output, KernelParams params) {
  const char *where = "token_logprob_hip_backward";
  const Tensor *x = inputs[0];
  if (x && !x->requires_grad) return;
  if (x && !x->grad) {
    report_error(where, "x requires a gradient but has none");
    return;
  }
  TokenArgs A;
  if (!token_args(A, x, x ? x->grad : nullptr, inputs[1], params.fval, where) ||
      !token_vectors(A, inputs[2], inputs[3], output, where) ||
      !upstream(output->grad, A.rows, &A.dlogp, where) ||
      !upstream(inputs[3]->grad, A.rows, &A.dentropy, where))
    return;
  if (A.rows == 0 || !ensure_init()) return;
  launch_backward(A, x->dtype, params.keepdim != 1);
  finish(where);
}

void token_logprob_step_hip(const Tensor *x, const Tensor *tokens, const Tensor *dlogp,
                            const Tensor *dentropy, Tensor *logp, Tensor *entropy, Tensor *dx,
                            float temperature) {
  const char *where = "token_logprob_step_hip";
  if (!dx) {
    report_error(where, "dx is NULL");
    return;
  }
  TokenArgs A;
  if (!token_args(A, x, dx, tokens, temperature, where)) return;
  const uint64_t N = A.rows;
  if (!f32_vector(entropy, N) || !f32_vector(logp, N)) {
    report_error(where, "entropy and logp must be contiguous FLOAT32 GPU tensors of %llu elements",
                 (unsigned long long)N);
    return;
  }
  A.entropy = static_cast<float *>(entropy->data);
  A.logp = static_cast<float *>(logp->data);
  if (!upstream(dlogp, N, &A.dlogp, where) || !upstream(dentropy, N, &A.dentropy, where) || N == 0 ||
      !ensure_init())
    return;
  A.stats = static_cast<float *>(partials(2 * N * sizeof(float), where));
  if (!A.stats) return;
  launch_forward(A, x->dtype);
  launch_backward(A, x->dtype, false);
  finish(where);
}

}  // extern "C"
