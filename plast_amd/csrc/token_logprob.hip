// token_logprob.hip — log-probabilities of given tokens with the rows' entropies, their most likely
// alternatives, and the gradient; the distribution of a row is p = softmax(x / T).
//
// The mathematics is in base 2, the hardware's exponential. With c = log2(e) / T, m the row's largest
// logit and z_j = c x_j - c m:
//   s = sum_j 2^z_j,  w = sum_j 2^z_j z_j,
//   log p_j = (x_j - m) / T - ln2 log2 s,  H = -sum_j p_j log p_j = ln2 (log2 s - w / s).
// c m is rounded once and z_j = fma(c, x_j, -c m) once more: the first rounding, r = c m - round(c m),
// moves every z_j alike, so p and H do not see it, and log p takes it out of log2 s again; the second is
// relative to z_j itself. r is at most half a step of c m: up to |c m| = kReach it is within 4 and 2^z_j in range;
// beyond it z_j = c (x_j - m), whose difference is rounded relative to itself and r is 0.
// Gradient for upstream u of log p[token] and h of H:
//   dx_j = (u ([j = token] - p_j) - h p_j (log p_j + H)) / T
//        = u / T [j = token] - 2^z_j (A + B z_j),
//   B = h ln2 / (T s),  A = (u + h H) / (T s) - B log2 s.
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "rows.hpp"

namespace plast {
namespace {

constexpr float kLn2 = 0.693147180559945309f;
constexpr float kInf = __builtin_huge_valf();
constexpr int kRowBlock = 256;  // lanes of a workgroup
// |c m| up to which c m and its rounding are used: a mask of -1e30 that a lane meets first, or that fills a row, has
// an r of 1e22, and 2^r is no number. 2^27 leaves logits of 20 a temperature of 2.2e-7.
constexpr float kReach = 0x1p27f;

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
  uint32_t first_row, rows, vocab;  // first_row: of a launch, where one cannot hold all
  float c;      // log2(e) / T
  float inv_t;  // 1 / T
  RowMap<2> map;  // of x and of its gradient
};

// The exponent z of a logit. Where c m is beyond kReach, c (x - m) is taken instead.
struct RowRef {
  float c, m, cm;
  bool far;
  __device__ __forceinline__ RowRef(float c_, float m_) : c(c_), m(m_), cm(c_ * m_) {
    far = !(fabsf(cm) < kReach);
  }
  __device__ __forceinline__ float z(float x) const {
    return far ? (x - m) * c : __builtin_fmaf(x, c, -cm);
  }
  // What the rounding of c m adds to every z.
  __device__ __forceinline__ float shift() const { return far ? 0.0f : __builtin_fmaf(c, m, -cm); }
};

// A unit's sum by pairs: beside a largest term of 1, the fewer roundings the better.
template <class F>
__device__ __forceinline__ float unit_sum(F f) {
  if constexpr (sizeof(F) == 32) return ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
  else return (f[0] + f[1]) + (f[2] + f[3]);
}
// The largest of a unit, NaN if one is.
template <class F>
__device__ __forceinline__ float unit_max(F f) {
  constexpr int E = sizeof(F) / sizeof(float);
  float g = f[0];
#pragma unroll
  for (int e = 1; e + 1 < E; e += 2) g = __builtin_elementwise_maximum(__builtin_elementwise_maximum(g, f[e]), f[e + 1]);
  return __builtin_elementwise_maximum(g, f[E - 1]);
}

// A lane's share of s and w, against a reference of its own that grows with the logits it meets: cm is
// c times the largest so far, but at least -kReach (a row whose largest logit is not in range is worked out by
// the exact path below).
struct Running {
  float m = -kInf, cm = -kReach, s = 0.0f, w = 0.0f;
  __device__ __forceinline__ void refer(float to) {
    const float d = cm - to, f = __builtin_amdgcn_exp2f(d);
    w = f * __builtin_fmaf(d, s, w);
    s *= f;
    cm = to;
  }
  __device__ __forceinline__ void grow(float c, float g) {
    m = __builtin_elementwise_maximum(m, g);  // NaN stays
    refer(fmaxf(c * m, -kReach));
  }
  // A logit's term, which the caller adds to s.
  __device__ __forceinline__ float term(float c, float x) {
    // below 2^-200 nothing is added, and a masked logit's -inf meets no 0
    const float z = fmaxf(__builtin_fmaf(x, c, -cm), -200.0f);
    const float e = __builtin_amdgcn_exp2f(z);
    w = __builtin_fmaf(e, z, w);
    return e;
  }
};
__device__ __forceinline__ Running wave_join(Running r) {
  float m = r.m, cm = r.cm;
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    m = __builtin_elementwise_maximum(m, __shfl_xor(m, d));
    cm = fmaxf(cm, __shfl_xor(cm, d));
  }
  r.refer(cm);
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    r.s += __shfl_xor(r.s, d);
    r.w += __shfl_xor(r.w, d);
  }
  r.m = m;
  return r;
}
// Whether the running form holds for a row with this largest logit.
__device__ __forceinline__ bool in_range(float c, float m) { return m == -kInf || fabsf(c * m) < kReach; }

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

__device__ __forceinline__ void put_stats(const TokenArgs &A, uint32_t row, float m, float l0) {
  if (!A.stats) return;  // the step keeps none
  A.stats[2 * row] = m;
  A.stats[2 * row + 1] = l0;
}

// The row's results, by one lane. s and w are over the whole row; `shift` is what every z holds beside c (x - m).
// l0, log2 of s / 2^shift, may be given.
__device__ __forceinline__ void row_out(const TokenArgs &A, uint32_t row, int32_t token, float x_token,
                                        float m, float s, float w, float shift, const float *exact_l0 = nullptr) {
  if (m == -kInf) {  // no logit that is not -inf
    A.logp[row] = uint32_t(token) < A.vocab ? -kInf : __builtin_nanf("");
    A.entropy[row] = 0.0f;
    put_stats(A, row, -kInf, 0.0f);
    return;
  }
  const float l0 = exact_l0 ? *exact_l0 : log2f(s) - shift;
  const float h = kLn2 * ((l0 + shift) - w / s);
  A.logp[row] = uint32_t(token) < A.vocab ? log_p(A, x_token, m, l0) : __builtin_nanf("");
  A.entropy[row] = h < 0.0f ? 0.0f : h;
  put_stats(A, row, m, l0);
}

__device__ __forceinline__ void pad_out(const TokenArgs &A, uint32_t row) {
  A.logp[row] = 0.0f;
  A.entropy[row] = 0.0f;
  put_stats(A, row, -kInf, 0.0f);
}

// ------------------------------------------------------------------------- forward

constexpr uint32_t kList = 256;  // candidates that are kept while a row is read

// What the W waves that share a row hold in LDS.
template <int W>
struct RowLds {
  float red[W][4];
  uint64_t keys[W];
  float group[64];
  float threshold;
  uint32_t count[2], ties;
  uint64_t list[2 * kList];  // two lists, or one where pieces are joined
};

__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
template <int W>
__device__ __forceinline__ void row_sync() {
  if constexpr (W == 1) wave_sync();
  else __syncthreads();
}

__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t k = uint32_t(key >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// An alternative at its place, by one lane; no key: the row is shorter than its alternatives.
__device__ __forceinline__ void put_top(const TokenArgs &A, uint32_t row, uint32_t k, uint64_t key, float m, float l0) {
  const uint64_t at = uint64_t(row) * A.top + k;
  A.top_ids[at] = key ? int32_t(0xffffffffu - uint32_t(key)) : -1;
  A.top_logp[at] = key ? log_p(A, key_value(key), m, l0) : -kInf;
}

// The sums of a row with NaN, infinite or out-of-range logits, whose largest logit m the one pass has found (NaN
// if one is): another pass, against m itself. Leaves m and l0, writes the row's results.
template <class T, int W>
__device__ __forceinline__ void exact_sums(const TokenArgs &A, const T *x, uint32_t row, int32_t token, float x_token,
                                           uint32_t gl, RowLds<W> &L, float &m, float &l0) {
  constexpr uint32_t NL = 64 * W;
  const uint32_t V = A.vocab;
  const RowRef ref(A.c, m);
  float s = 0.0f, w = 0.0f;
  for (uint32_t j = gl; j < V; j += NL) {
    const float z = ref.z(float(x[j])), e = __builtin_amdgcn_exp2f(z);
    s += e;  // NaN for a NaN or a +inf logit
    w = __builtin_fmaf(e, fmaxf(z, -FLT_MAX), w);
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) {
    s += __shfl_xor(s, d);
    w += __shfl_xor(w, d);
  }
  if constexpr (W > 1) {
    row_sync<W>();
    if (gl % 64 == 0) L.red[gl / 64][0] = s, L.red[gl / 64][1] = w;
    row_sync<W>();
    s = L.red[0][0], w = L.red[0][1];
    for (int k = 1; k < W; ++k) s += L.red[k][0], w += L.red[k][1];
  }
  if (s != s) m = s;
  l0 = log2f(s) - ref.shift();
  if (gl == 0) row_out(A, row, token, x_token, m, s, w, ref.shift());
}

// The alternatives of a row with NaN or infinite logits, or of one that the list could not hold in the end: an argmax
// each, a pass over the row.
template <class T, int W>
__device__ __forceinline__ void exact_top(const TokenArgs &A, const T *x, uint32_t row, uint32_t gl, RowLds<W> &L, float m,
                                          float l0) {
  constexpr uint32_t NL = 64 * W;
  const uint32_t V = A.vocab, wave = gl / 64;
  uint64_t last = 0;
  for (uint32_t k = 0; k < A.top; ++k) {
    uint64_t best = 0;
    for (uint32_t j = gl; j < V; j += NL) {
      const uint64_t key = order_key(float(x[j]), j);
      if ((k == 0 || key < last) && key > best) best = key;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      const uint64_t o = __shfl_xor((unsigned long long)best, d);
      best = o > best ? o : best;
    }
    row_sync<W>();
    if (gl % 64 == 0) L.keys[wave] = best;
    row_sync<W>();
    for (int d = 0; d < W; ++d) best = L.keys[d] > best ? L.keys[d] : best;
    if (gl == 0) {
      put_top(A, row, k, best, m, l0);
      if (best && uint32_t(best >> 32) == 0xffffffffu) A.top_logp[uint64_t(row) * A.top + k] = __builtin_nanf("");
    }
    last = best;
  }
}

// Finds the `top` largest logits of a row while it is read, by units: a unit's key is its largest logit and its
// number, and the largest logits all lie in the `top` units of the largest keys (a logit of another unit has
// `top` logits before it, those units' largest). A bound under which no unit counts starts as the top-th
// largest of 16, 32 or 64 lane groups' maxima over the first logits, twice `top` groups at least, and is raised to
// the top-th unit whenever as many logits again have been read; only units above it go to the list, some
// top ln(units) in all where the logits are in no order. Where they rise, or the first batch is masked and a later one is
// not, a batch has more units above the bound than the list holds: the row is given up, and read twice more when its end
// is reached ([4096, 32000] in fp32 with 5 86 us, 207 if a start of each row is masked; [4096, 131072] in bf16 with 8 182
// and 450). Lists of the waves' own, which never overflow as each batch bounds its units first, cost 234 there, but
// 216 where there is no order. Logits after the last whole unit are units of their own.
template <class T, int W>
struct Candidates {
  static constexpr uint32_t NL = 64 * W, E = Unit<T>::E;
  RowLds<W> &L;
  const T *x;
  uint32_t gl, top, units, cur = 0;
  float bound = kInf;  // units above it are candidates
  bool lost = false;   // the list was too short
  uint32_t held = 0;   // its length, where a wave has its own
  __device__ __forceinline__ Candidates(RowLds<W> &l, const T *row, uint32_t g, uint32_t t, uint32_t n)
      : L(l), x(row), gl(g), top(t), units(n) {}

  // By whole waves: the lanes that `hot` names add theirs.
  __device__ __forceinline__ void push(bool hot, float v, uint32_t number) {
    const uint64_t hits = __ballot(hot);
    if (!hits) return;
    const uint32_t n = __popcll(hits), before = __popcll(hits & ((uint64_t(1) << (gl & 63)) - 1));
    uint32_t at = held;
    if constexpr (W == 1) {
      held += n;
    } else {
      if ((gl & 63) == 0) at = atomicAdd(&L.count[cur], n);
      at = __builtin_amdgcn_readfirstlane(at);
    }
    if (hot && at + before < kList) L.list[cur * kList + at + before] = order_key(v, number);
  }
  __device__ __forceinline__ uint32_t listed() const { return W == 1 ? held : L.count[cur]; }
  __device__ __forceinline__ void relist(uint32_t n, uint32_t list) {
    if constexpr (W == 1) held = n;
    else if (gl == 0) L.count[list] = n;
  }
  __device__ __forceinline__ void clear() {
    if (gl == 0) L.count[0] = L.count[1] = L.ties = 0;
  }
  // The bound from every lane's maximum over the first logits; clear() comes before it.
  __device__ __forceinline__ void start(float lane_max) {
    float v = lane_max;
    if constexpr (W > 1) {
#pragma unroll
      for (int d = W / 2; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
      if (gl % W == 0) L.group[gl / W] = v;
      row_sync<W>();
      v = L.group[gl % 64];
    } else {
      row_sync<W>();
    }
    uint32_t before = 0;
    const auto count = [&](auto groups) {
      constexpr uint32_t G = decltype(groups)::value;
#pragma unroll
      for (uint32_t d = 32; d >= G; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
#pragma unroll
      for (uint32_t d = 0; d < G; ++d) before += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), d)) > v;
    };
    if (top <= 8) count(std::integral_constant<uint32_t, 16>{});
    else if (top <= 16) count(std::integral_constant<uint32_t, 32>{});
    else count(std::integral_constant<uint32_t, 64>{});
    // the top-th largest: the smallest that fewer than `top` exceed
    v = before < top ? v : kInf;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v = fminf(v, __shfl_xor(v, d));
    bound = v;
  }
  // After start()'s logits: the units above the bound are in the list and `equal` counts this lane's at it. The
  // lowest of the equal ones are found by rereading the units from..to and the tail where there are many (a
  // mask).
  template <class F>
  __device__ __forceinline__ void take_equal(uint32_t equal, F &&push_equal, uint32_t from, uint32_t to, uint32_t tail) {
    if (equal) atomicAdd(&L.ties, equal);
    row_sync<W>();
    const uint32_t above = listed(), ties = L.ties;
    row_sync<W>();
    if (above > kList) {
      give_up();
      return;
    }
    if (above >= top || ties == 0) return;
    if (above + ties <= kList) {
      push_equal();
      row_sync<W>();
      return;
    }
    uint32_t want = top - above, at = above;
    if (gl < 64)
      for (uint32_t n0 = from; want && n0 < to + tail; n0 += 64) {
        const uint32_t n = n0 + gl;
        float v = __builtin_nanf("");
        if (n < to) v = unit_max(to_floats<T>(load_unit(x + uint64_t(n) * E)));
        else if (n < to + tail) v = float(x[uint64_t(to) * E + (n - to)]);
        const uint64_t hit = __ballot(v == bound);
        const uint32_t place = __popcll(hit & ((uint64_t(1) << gl) - 1));
        if (v == bound && place < want) L.list[at + place] = order_key(v, n);
        const uint32_t got = min(uint32_t(__popcll(hit)), want);
        want -= got;
        at += got;
      }
    relist(at, 0);
    row_sync<W>();
  }
  __device__ __forceinline__ void give_up() {
    lost = true;
    bound = kInf;
  }
  // The place of a candidate among the list's n.
  __device__ __forceinline__ uint32_t rank(uint64_t key, uint32_t n) const {
    uint32_t r = 0;
#pragma unroll 4
    for (uint32_t k = 0; k < n; ++k) r += L.list[cur * kList + k] > key;
    return r;
  }
  // Drops all but the `top` largest and raises the bound to the last of them.
  __device__ __forceinline__ void raise() {
    row_sync<W>();
    const uint32_t n = listed();
    if (n > kList) give_up();
    if (lost || n <= top) {
      row_sync<W>();
      return;
    }
    for (uint32_t i = gl; i < n; i += NL) {
      const uint64_t key = L.list[cur * kList + i];
      const uint32_t r = rank(key, n);
      if (r < top) L.list[(1 - cur) * kList + r] = key;
      if (r == top - 1) L.threshold = key_value(key);
    }
    relist(top, 1 - cur);
    cur = 1 - cur;
    row_sync<W>();
    bound = L.threshold;
  }
  // Batches of the units from..to, for all lanes: f(unit's number, whether there is one, its largest logit).
  template <class F>
  __device__ __forceinline__ void each_unit(uint32_t from, uint32_t to, F &&f) const {
    constexpr uint32_t U = W == 1 ? 1 : 2;  // more would take more registers than the first pass
    for (uint32_t q0 = from; q0 < to; q0 += NL * U) {
      typename Unit<T>::vec v[U];
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) {
        const uint32_t q = q0 + u * NL + gl;
        if (q < to) v[u] = load_unit(x + uint64_t(q) * E);
      }
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) {
        const uint32_t q = q0 + u * NL + gl;
        f(q, q < to, q < to ? unit_max(to_floats<T>(v[u])) : 0.0f);
      }
    }
  }
  // The list of a row that was given up, by two more passes: the units at or above the top-th largest of 64 groups'
  // largest keys, which has `top` units at or above it. Neighbours are in different groups, so that of units which stand
  // together few more than `top` are left. More than the list holds are left where many of the largest are 64 or a
  // multiple apart: that row stays given up.
  __device__ __forceinline__ void reread(uint32_t from, uint32_t to, uint32_t tails) {
    const bool has_tail = gl < tails;
    const float tail = has_tail ? float(x[units * E + gl]) : 0.0f;
    const uint64_t tail_key = has_tail ? order_key(tail, units + gl) : 0;
    uint64_t key = tail_key, *const group = L.list + kList;
    each_unit(from, to, [&](uint32_t q, bool is, float v) {
      const uint64_t k = order_key(v, q);
      if (is && k > key) key = k;
    });
    row_sync<W>();
    if (gl < 64) group[gl] = 0;
    row_sync<W>();
    atomicMax(reinterpret_cast<unsigned long long *>(&group[gl % 64]), (unsigned long long)key);
    row_sync<W>();
    key = group[gl % 64];
    uint32_t before = 0;
#pragma unroll 4
    for (uint32_t k = 0; k < 64; ++k) before += group[k] > key;
    const uint64_t last = __ballot(key && before == top - 1);  // none: fewer than `top` units, all of them count
    uint64_t least = 0;
    if (last) {
      const int lane = __ffsll((unsigned long long)last) - 1;
      least = uint64_t(uint32_t(__builtin_amdgcn_readlane(uint32_t(key >> 32), lane))) << 32 |
              uint32_t(__builtin_amdgcn_readlane(uint32_t(key), lane));
    }
    cur = 0;
    relist(0, 0);
    row_sync<W>();
    each_unit(from, to, [&](uint32_t q, bool is, float v) { push(is && order_key(v, q) >= least, v, q); });
    push(has_tail && tail_key >= least, tail, units + gl);
    row_sync<W>();
    bound = key_value(least);
    lost = listed() > kList;
    row_sync<W>();
  }
  // The units' logits in their place: the list holds logits from here on.
  __device__ __forceinline__ void open(uint32_t from, uint32_t to, uint32_t tails) {
    raise();
    if (lost) {
      reread(from, to, tails);
      if (lost) return;
      raise();
    }
    const uint32_t n = listed(), old = cur;
    const float least = n == top ? bound : -kInf;  // the top-th logit is no smaller
    row_sync<W>();
    cur = 1 - cur;
    relist(0, cur);
    row_sync<W>();
    for (uint32_t i0 = 0; i0 < n * E; i0 += NL) {
      const uint32_t i = i0 + gl;
      bool hot = i < n * E;
      float v = 0.0f;
      uint32_t j = 0;
      if (hot) {
        const uint32_t number = 0xffffffffu - uint32_t(L.list[old * kList + i / E]), e = i % E;
        j = number < units ? number * E + e : units * E + (number - units);
        hot = number < units || e == 0;
        v = float(x[j]);
        hot = hot && v >= least;
      }
      push(hot, v, j);
    }
    row_sync<W>();
  }
};

// A piece of a row, where rows are cut because there are few: what it found, for the last to finish.
struct Piece {
  float m, cm, s, w;
  uint64_t keys[PLAST_TOP_MAX];
  uint32_t lost;  // the list was too short
};
struct Pieces {
  uint32_t n, r, q;
  Piece *found;  // [rows][n]
};
constexpr uint32_t kMaxPieces = 32, kCutBlocks = 512;  // of a row, of a launch
// What bounds a row's candidates among its n pieces' keys: the q-th largest of the pieces' r-th keys, q r >= top, which
// has `top` keys at or above it. Of independent logits some three times `top` are, where the largest of the last keys
// leaves nearly all of them, more than a list holds ([1, 131072] in fp32 with 20: 1468 us, the row read again for each).
// In any row the q pieces leave at most `top` each and the others r - 1. Finding it takes a step a piece: where there are
// as many pieces as keys of each, and few keys in all, the largest of the last ones will do ([1, 131072] in fp32 with 5
// 11.3 us and 11.8, [64, 50001] in fp16 with 5 12.0 and 12.4; but [64, 131072] in bf16 with 20 20.1 and 19.0, [1, 131072] in
// fp32 with 10 12.9 and 12.4).
constexpr uint32_t bound_key(uint32_t top, uint32_t n) {
  const uint32_t r = (3 * top + n - 1) / n;
  return r < top && (top > n || top * n > 192) ? r : top;
}
constexpr bool joined_keys_fit() {
  for (uint32_t top = 1; top <= PLAST_TOP_MAX; ++top)
    for (uint32_t n = 2; n <= kMaxPieces; ++n) {
      const uint32_t r = bound_key(top, n), q = (top + r - 1) / r;
      if (q > n || q * top + (n - q) * (r - 1) > 2 * kList) return false;
    }
  return true;
}
static_assert(joined_keys_fit(), "the pieces' keys that count fit both lists");
__device__ uint32_t g_tickets[kCutBlocks / 2];  // of each row, zero between launches

// W waves per row (or piece of one), four rows per workgroup where W is 1. One pass: a lane's units of 16 bytes
// come four at a time. What bounds it is the read for fp32 ([8184, 32000] 143 us, 6.5 TB/s, vector units 44% busy) and the
// vector units, with the read close behind, for the 16-bit types, whose logit takes ten issue slots, four of them the
// exponential's, as fp32's does ([8192, 49999] in bf16 124 us, 78% busy; [4096, 131072] with 8 alternatives 182 us, 83%).
// With alternatives a lane may have 64 registers, so that eight waves share a SIMD (with 77, 203 us).
template <class T, int W, bool TOP, bool CUT>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W, TOP ? 8 : 1) void fwd_kernel(TokenArgs A, Pieces P) {
  constexpr uint32_t NL = 64 * W, E = Unit<T>::E, U = 4;
  __shared__ RowLds<W> lds[W == 1 ? 4 : 1];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t gl = W == 1 ? threadIdx.x & 63 : threadIdx.x;
  RowLds<W> &L = lds[W == 1 ? wave : 0];
  const uint32_t local = W == 1 ? blockIdx.x * 4 + wave : CUT ? blockIdx.x / P.n : blockIdx.x;
  const uint32_t row = A.first_row + local;
  const uint32_t piece = CUT ? blockIdx.x - local * P.n : 0, pieces = CUT ? P.n : 1;
  if (W == 1 && local >= A.rows) return;
  const int32_t token = A.tokens[row];
  const uint32_t V = A.vocab, units = V / E;
  const T *x = static_cast<const T *>(A.x) + row_at(A.map, row).at[0];
  const uint32_t from = uint32_t(uint64_t(units) * piece / pieces), to = uint32_t(uint64_t(units) * (piece + 1) / pieces);
  // where rows are few, their first units are on their way before the token is known
  typename Unit<T>::vec v[U];
  const auto fetch = [&](uint32_t q0) {
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t q = q0 + u * NL + gl;
      if (q < to) v[u] = load_unit(x + uint64_t(q) * E);
    }
  };
  if constexpr (W > 1) fetch(from);
  if (token < 0) {
    if (piece == 0) {
      if (gl == 0) pad_out(A, row);
      if (TOP && gl < A.top) put_top(A, row, gl, 0, 0.0f, 0.0f);
    }
    return;
  }
  const float x_token = uint32_t(token) < V ? float(x[token]) : 0.0f;
  // the logits after the last unit, one a lane
  const bool has_tail = piece == pieces - 1 && gl < V - units * E;
  const float tail = has_tail ? float(x[units * E + gl]) : -kInf;
  const bool tail_first = to - from <= NL * U;  // then it is among the first logits
  const float c = A.c;
  Running r;
  Candidates<T, W> top(L, x, gl, A.top, units);
  if constexpr (TOP) top.clear();
  uint32_t batch = 0;
  uint32_t q0 = from;
  do {
    if (W == 1 || batch) fetch(q0);
    float most = tail_first ? tail : -kInf;
    float largest[U];  // of each unit
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t q = q0 + u * NL + gl;
      largest[u] = -kInf;
      if (q >= to) continue;
      const auto f = to_floats<T>(v[u]);
      const float g = unit_max(f);
      if (!(g <= r.m)) r.grow(c, g);
      auto terms = f;
#pragma unroll
      for (uint32_t e = 0; e < E; ++e) terms[e] = r.term(c, f[e]);
      r.s += unit_sum(terms);
      if constexpr (TOP) {
        largest[u] = g;
        most = fmaxf(most, g);
      }
    }
    if constexpr (TOP) {
      if (batch == 0) {
        top.start(most);
        const bool tail_now = tail_first && has_tail;
        uint32_t equal = tail_now && tail == top.bound;
        top.push(tail_now && tail > top.bound, tail, units + gl);
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
          const uint32_t q = q0 + u * NL + gl;
          top.push(largest[u] > top.bound, largest[u], q);
          equal += q < to && largest[u] == top.bound;
        }
        top.take_equal(
            equal,
            [&] {
              top.push(tail_now && tail == top.bound, tail, units + gl);
#pragma unroll
              for (uint32_t u = 0; u < U; ++u) {
                const uint32_t q = q0 + u * NL + gl;
                top.push(q < to && largest[u] == top.bound, largest[u], q);
              }
            },
            from, min(q0 + NL * U, to), tail_first && piece == pieces - 1 ? V - units * E : 0);
      } else {
        if (__any(most > top.bound))
#pragma unroll
          for (uint32_t u = 0; u < U; ++u) top.push(largest[u] > top.bound, largest[u], q0 + u * NL + gl);
        if (((batch + 1) & batch) == 0 || (W == 1 && top.listed() > kList / 2)) top.raise();
      }
    }
    ++batch;
    q0 += NL * U;
  } while (q0 < to);
  if (has_tail) {
    if (!(tail <= r.m)) r.grow(c, tail);
    r.s += r.term(c, tail);
  }
  if (TOP && !tail_first) top.push(has_tail && tail > top.bound, tail, units + gl);
  r = wave_join(r);
  if constexpr (W > 1) {
    if (gl % 64 == 0) {
      L.red[gl / 64][0] = r.m;
      L.red[gl / 64][1] = r.cm;
      L.red[gl / 64][2] = r.s;
      L.red[gl / 64][3] = r.w;
    }
    __syncthreads();
    r.m = L.red[0][0], r.cm = L.red[0][1], r.s = L.red[0][2], r.w = L.red[0][3];
    for (int k = 1; k < W; ++k) {
      Running o;
      o.m = L.red[k][0], o.cm = L.red[k][1], o.s = L.red[k][2], o.w = L.red[k][3];
      const float cm = fmaxf(r.cm, o.cm);
      r.refer(cm);
      o.refer(cm);
      r.m = __builtin_elementwise_maximum(r.m, o.m);
      r.s += o.s;
      r.w += o.w;
    }
  } else {
    row_sync<W>();
  }
  uint32_t found = 0;
  if constexpr (TOP) {
    top.open(from, to, piece == pieces - 1 ? V - units * E : 0);
    found = top.listed();
  }
  if constexpr (CUT) {
    __shared__ bool is_last;
    Piece *mine = P.found + uint64_t(row) * P.n;
    if (gl == 0) {
      put_shared(&mine[piece].m, r.m);
      put_shared(&mine[piece].cm, r.cm);
      put_shared(&mine[piece].s, r.s);
      put_shared(&mine[piece].w, r.w);
      put_shared(&mine[piece].lost, uint32_t(top.lost));
    }
    if (TOP && !top.lost) {
      for (uint32_t i = gl; i < found; i += NL) {
        const uint64_t key = L.list[top.cur * kList + i];
        const uint32_t k = top.rank(key, found);
        if (k < A.top) put_shared(&mine[piece].keys[k], key);
      }
      if (gl >= found && gl < A.top) put_shared(&mine[piece].keys[gl], uint64_t(0));
    }
    // every wave's stores have reached the memory that the XCDs share before the ticket is drawn
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (gl == 0)
      is_last = __hip_atomic_fetch_add(&g_tickets[row], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == P.n - 1;
    __syncthreads();
    if (!is_last) return;
    if (gl == 0) put_shared(&g_tickets[row], 0u);
    // a wave's lanes take the pieces; the merged sums are the same whoever comes last
    Running o;
    const uint32_t lane = gl % 64;
    uint32_t lost = 0;
    uint64_t mid = 0, keys[kMaxPieces * PLAST_TOP_MAX / NL];
    if (lane < P.n) {
      o.m = get_shared(&mine[lane].m), o.cm = get_shared(&mine[lane].cm);
      o.s = get_shared(&mine[lane].s), o.w = get_shared(&mine[lane].w);
      if constexpr (TOP) {
        lost = get_shared(&mine[lane].lost);
        mid = get_shared(&mine[lane].keys[P.r - 1]);
      }
    }
    if constexpr (TOP) {
#pragma unroll
      for (uint32_t t = 0; t < kMaxPieces * PLAST_TOP_MAX / NL; ++t) {
        const uint32_t i = gl + t * NL, p = i / A.top;
        keys[t] = p < P.n ? get_shared(&mine[p].keys[i - p * A.top]) : 0;
      }
    }
    r = wave_join(o);
    top.lost = __any(lost != 0);
    if (TOP && !top.lost) {
      uint64_t least = mid;
      const bool one = P.q == 1;
      if (!one) {
        uint32_t before = 0;
        for (uint32_t k = 0; k < P.n; ++k) {
          const uint32_t high = __builtin_amdgcn_readlane(uint32_t(mid >> 32), k);
          before += (uint64_t(high) << 32 | uint32_t(__builtin_amdgcn_readlane(uint32_t(mid), k))) > mid;
        }
        if (before >= P.q) least = ~uint64_t(0);
      }
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) {
        const uint64_t k = __shfl_xor((unsigned long long)least, d);
        least = (k > least) == one ? k : least;
      }
      top.cur = 0;
      if (gl == 0) L.count[0] = 0;
      __syncthreads();
#pragma unroll
      for (uint32_t t = 0; t < kMaxPieces * PLAST_TOP_MAX / NL; ++t)
        if (keys[t] >= least && keys[t]) L.list[atomicAdd(&L.count[0], 1u)] = keys[t];
      __syncthreads();
      found = L.count[0];
    }
  }
  float m = r.m, l0;
  if (!in_range(c, m)) {
    exact_sums<T, W>(A, x, row, token, x_token, gl, L, m, l0);
  } else {
    const float shift = RowRef(c, m).shift();
    l0 = log2f(r.s) - shift;
    if (gl == 0) row_out(A, row, token, x_token, m, r.s, r.w, shift);
  }
  if constexpr (TOP) {
    if (m != m || top.lost) {
      exact_top<T, W>(A, x, row, gl, L, m, l0);
      return;
    }
    for (uint32_t i = gl; i < found; i += NL) {
      const uint64_t key = L.list[top.cur * kList + i];
      const uint32_t k = top.rank(key, found);
      if (k < A.top) put_top(A, row, k, key, m, l0);
    }
    if (gl >= found && gl < A.top) put_top(A, row, gl, 0, m, l0);
  }
}

// ------------------------------------------------------------------------- backward

// A row's gradient: dx = onehot - 2^z (a + b z).
struct RowGrad {
  RowRef ref;
  float a, b, onehot;
  __device__ __forceinline__ RowGrad(const TokenArgs &A, uint32_t row, int32_t token, float m, float l, float entropy)
      : ref(A.c, m) {
    const float u = A.dlogp ? A.dlogp[row] : 0.0f, h = A.dentropy ? A.dentropy[row] : 0.0f;
    const float r = A.inv_t * __builtin_amdgcn_exp2f(-l);  // 1 / (T s)
    b = h * kLn2 * r;
    a = uint32_t(token) < A.vocab ? (u + h * entropy) * r - b * l : __builtin_nanf("");
    onehot = u * A.inv_t;
  }
  __device__ __forceinline__ float at(float x) const {
    const float z = fmaxf(ref.z(x), -200.0f);  // 2^-200 is 0, and a masked logit's z stays finite
    return -__builtin_amdgcn_exp2f(z) * __builtin_fmaf(b, z, a);
  }
};

// A row in units that start at 16-byte boundaries of its gradient, where the stores go (the reads take any
// address): unit q holds elements first .. first + E - 1, of which those inside the row count.
template <class T>
struct RowUnits {
  static constexpr uint32_t E = Unit<T>::E;
  int32_t shift;
  uint32_t V;
  __device__ __forceinline__ RowUnits(const T *g, uint32_t v)
      : shift(int32_t(uint32_t(reinterpret_cast<uintptr_t>(g) / sizeof(T)) % E)), V(v) {}
  __device__ __forceinline__ int32_t first(uint32_t q) const { return int32_t(q * E) - shift; }
  __device__ __forceinline__ bool whole(int32_t j) const { return j >= 0 && j + int32_t(E) <= int32_t(V); }
  // A unit's elements; those outside the row are -inf.
  __device__ __forceinline__ typename Unit<T>::vec load(const T *x, int32_t j) const {
    if (whole(j)) return load_unit(x + j);
    typename Unit<T>::vec v;
#pragma unroll
    for (int32_t e = 0; e < int32_t(E); ++e) v[e] = j + e >= 0 && j + e < int32_t(V) ? x[j + e] : T(-kInf);
    return v;
  }
  template <bool ADD>
  __device__ __forceinline__ void store(T *g, int32_t j, typename Unit<T>::floats f) const {
    if (whole(j)) {
      typename Unit<T>::vec *to = reinterpret_cast<typename Unit<T>::vec *>(g + j);
      if constexpr (ADD) f += to_floats<T>(__builtin_nontemporal_load(to));
      __builtin_nontemporal_store(__builtin_convertvector(f, typename Unit<T>::vec), to);
      return;
    }
#pragma unroll
    for (int32_t e = 0; e < int32_t(E); ++e)
      if (j + e >= 0 && j + e < int32_t(V)) g[j + e] = T(ADD ? f[e] + float(g[j + e]) : f[e]);
  }
};
// Units of the longest row of v elements, whatever its address.
template <class T>
constexpr uint32_t most_units(uint32_t v) {
  return (v + 2 * (Unit<T>::E - 1)) / Unit<T>::E;
}

template <class T, bool ADD>
__device__ __forceinline__ void grad_unit(const RowUnits<T> &R, const RowGrad &G, const T *x, T *dx, int32_t token,
                                          int32_t j) {
  auto f = to_floats<T>(R.load(x, j));
#pragma unroll
  for (int32_t e = 0; e < int32_t(R.E); ++e) {
    f[e] = G.at(f[e]);
    if (token == j + e) f[e] += G.onehot;
  }
  R.template store<ADD>(dx, j, f);
}

// Rows of many units: a workgroup takes BWD_UNITS units a lane of one row, whose constants are uniform.
constexpr uint32_t kBwdUnits = 2;
template <class T, bool ADD>
__global__ __launch_bounds__(kRowBlock) void bwd_kernel(TokenArgs A, uint32_t chunks) {
  const uint32_t block_row = blockIdx.x / chunks, row = A.first_row + block_row;
  const uint32_t q0 = (blockIdx.x - block_row * chunks) * kBwdUnits * kRowBlock + threadIdx.x;
  const int32_t token = A.tokens[row];
  const RowAt<2> at = row_at(A.map, row);
  T *dx = static_cast<T *>(A.dx) + at.at[1];
  const RowUnits<T> R(dx, A.vocab);
  const float m = A.stats[2 * row];
  if (token < 0 || m == -kInf) {
    if (ADD) return;
    typename Unit<T>::floats none = 0.0f;
#pragma unroll
    for (uint32_t u = 0; u < kBwdUnits; ++u) {
      const int32_t j = R.first(q0 + u * kRowBlock);
      if (j < int32_t(A.vocab)) R.template store<false>(dx, j, none);
    }
    return;
  }
  const T *x = static_cast<const T *>(A.x) + at.at[0];
  const RowGrad G(A, row, token, m, A.stats[2 * row + 1] + RowRef(A.c, m).shift(), A.entropy[row]);
#pragma unroll
  for (uint32_t u = 0; u < kBwdUnits; ++u) {
    const int32_t j = R.first(q0 + u * kRowBlock);
    if (j < int32_t(A.vocab)) grad_unit<T, ADD>(R, G, x, dx, token, j);
  }
}

// Short rows: one unit a lane, whatever rows a workgroup's lanes fall into.
template <class T, bool ADD>
__global__ __launch_bounds__(kRowBlock) void bwd_short_kernel(TokenArgs A, MagicDiv units) {
  const uint64_t at_unit = uint64_t(blockIdx.x) * kRowBlock + threadIdx.x;
  if (at_unit >= uint64_t(A.rows) * units.d) return;
  const uint32_t row = units.div(uint32_t(at_unit)), q = uint32_t(at_unit) - row * units.d;
  const int32_t token = A.tokens[row];
  const RowAt<2> at = row_at(A.map, row);
  T *dx = static_cast<T *>(A.dx) + at.at[1];
  const RowUnits<T> R(dx, A.vocab);
  const int32_t j = R.first(q);
  if (j >= int32_t(A.vocab)) return;
  const float m = A.stats[2 * row];
  if (token < 0 || m == -kInf) {
    typename Unit<T>::floats none = 0.0f;
    if (!ADD) R.template store<false>(dx, j, none);
    return;
  }
  const RowGrad G(A, row, token, m, A.stats[2 * row + 1] + RowRef(A.c, m).shift(), A.entropy[row]);
  grad_unit<T, ADD>(R, G, static_cast<const T *>(A.x) + at.at[0], dx, token, j);
}

// ------------------------------------------------------------------------- rows in registers

// The largest and the sum over the L lanes that share a row.
template <int L>
__device__ __forceinline__ float lanes_max(float v, float *lds) {
#pragma unroll
  for (int d = (L < 64 ? L : 64) / 2; d >= 1; d >>= 1) v = __builtin_elementwise_maximum(v, __shfl_xor(v, d));
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int k = 1; k < L / 64; ++k) v = __builtin_elementwise_maximum(v, lds[k]);
  }
  return v;
}
template <int L>
__device__ __forceinline__ float lanes_sum(float v, float *lds) {
#pragma unroll
  for (int d = (L < 64 ? L : 64) / 2; d >= 1; d >>= 1) v += __shfl_xor(v, d);
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int k = 1; k < L / 64; ++k) v += lds[k];
  }
  return v;
}

// log2 of s / 2^shift from the rest of s beside its `ones` largest terms of 2^shift each: log1p, rounded once where a
// sum around 1 would lose what a likely token's log p, close to 0, consists of.
__device__ __forceinline__ float log2_sum(float rest, float ones, float shift) {
  constexpr float kLog2e = 1.44269504088896341f;
  return log1pf(rest * __builtin_amdgcn_exp2f(-shift) + (ones - 1.0f)) * kLog2e;
}

// Forward and gradient (GRAD), or the forward alone, of rows that L lanes hold in N units each: one read, one
// write. Rows of up to a wave's lanes share workgroups. In short rows, where a likely token can have nearly all of
// the distribution, the largest logits' terms are counted apart from the others' sum (three instructions a logit: 14%
// of the step's time if the long rows had it too).
template <class T, int L, int N, bool GRAD>
__global__ __launch_bounds__(L > kRowBlock ? L : kRowBlock) void held_kernel(TokenArgs A) {
  constexpr uint32_t B = L > kRowBlock ? L : kRowBlock, E = Unit<T>::E;
  constexpr uint32_t ROWS = L > 64 ? 1 : B / L;
  static_assert(L <= 64 || L == B, "a row has a workgroup or lanes of a wave");
  constexpr bool APART = L <= 16;
  __shared__ float lds[3][16];
  const uint32_t V = A.vocab, gl = threadIdx.x % L;
  const uint32_t r = blockIdx.x * ROWS + threadIdx.x / L;
  const bool valid = ROWS == 1 || r < A.rows;
  const uint32_t row = A.first_row + (valid ? r : A.rows - 1);
  const int32_t token = A.tokens[row];
  const RowAt<2> at = row_at(A.map, row);
  const T *x = static_cast<const T *>(A.x) + at.at[0];
  T *dx = static_cast<T *>(A.dx) + at.at[1];
  const RowUnits<T> R(GRAD ? dx : x, V);
  typename Unit<T>::vec v[N];
  if (token >= 0) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int32_t j = R.first(u * L + gl);
      if (j < int32_t(V)) v[u] = R.load(x, j);
      else v[u] = T(-kInf);
    }
  } else {
#pragma unroll
    for (int u = 0; u < N; ++u) v[u] = T(-kInf);
  }
  const float x_token = gl == 0 && uint32_t(token) < V ? float(x[token]) : 0.0f;
  float m = -kInf;
#pragma unroll
  for (int u = 0; u < N; ++u) m = __builtin_elementwise_maximum(m, unit_max(to_floats<T>(v[u])));
  m = lanes_max<L>(m, lds[0]);
  const RowRef ref(A.c, m);
  const float ref_shift = ref.shift();
  float s = 0.0f, w = 0.0f;
  uint32_t ones = 0;
  if (m != -kInf) {
    const auto sums = [&](auto far) {
#pragma unroll
      for (int u = 0; u < N; ++u) {
        keep_raw(v[u]);
        const auto f = to_floats<T>(v[u]);
        auto terms = f;
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) {
          const float z = fmaxf(far ? (f[e] - m) * A.c : __builtin_fmaf(f[e], A.c, -ref.cm), -200.0f);
          const float p = __builtin_amdgcn_exp2f(z);
          if constexpr (APART) {
            ones += f[e] == m;
            terms[e] = f[e] == m ? 0.0f : p;
          } else {
            terms[e] = p;
          }
          w = __builtin_fmaf(p, z, w);
        }
        s += unit_sum(terms);
      }
    };
    if (ref.far) sums(std::true_type{});
    else sums(std::false_type{});
  }
  s = lanes_sum<L>(s, lds[1]);
  w = lanes_sum<L>(w, lds[2]);
  if (!(fabsf(m) <= FLT_MAX) && m != -kInf) m = __builtin_nanf("");  // a NaN or an infinite logit
  float l0;
  if constexpr (APART) {
    const float n = lanes_sum<L>(float(ones), nullptr);
    l0 = log2_sum(s, n, ref.shift());
    s += n * __builtin_amdgcn_exp2f(ref.shift());
  } else {
    l0 = log2f(s) - ref.shift();
  }
  if (m != m) l0 = m;
  if (gl == 0 && valid) {
    if (token < 0) pad_out(A, row);
    else row_out(A, row, token, x_token, m, s, w, ref.shift(), &l0);
  }
  if constexpr (GRAD) {
    if (!valid) return;
    if (m == -kInf) {  // padding too
      typename Unit<T>::floats none = 0.0f;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int32_t j = R.first(u * L + gl);
        if (j < int32_t(V)) R.template store<false>(dx, j, none);
      }
      return;
    }
    const float l = l0 + ref_shift, h = kLn2 * (l - w / s);
    const RowGrad G(A, row, token, m, l, h < 0.0f ? 0.0f : h);
    const auto grads = [&](auto far) {
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int32_t j = R.first(u * L + gl);
        if (j >= int32_t(V)) continue;
        keep_raw(v[u]);
        auto f = to_floats<T>(v[u]);
#pragma unroll
        for (int32_t e = 0; e < int32_t(E); ++e) {
          const float z = fmaxf(far ? (f[e] - m) * A.c : __builtin_fmaf(f[e], A.c, -ref.cm), -200.0f);
          f[e] = -__builtin_amdgcn_exp2f(z) * __builtin_fmaf(G.b, z, G.a);
          if (token == j + e) f[e] += G.onehot;
        }
        R.template store<false>(dx, j, f);
      }
    };
    if (ref.far) grads(std::true_type{});
    else grads(std::false_type{});
  }
}

// Alternatives of rows that a few lanes hold, one logit each: a logit's place is the number of those before it, counted
// by passing the keys round. [60000, 18] in fp32 with 5: 26 us, a wave a row and its list in LDS 47.
template <class T, int L>
__global__ __launch_bounds__(kRowBlock) void tiny_kernel(TokenArgs A) {
  const uint32_t gl = threadIdx.x % L, r = blockIdx.x * (kRowBlock / L) + threadIdx.x / L;
  const bool valid = r < A.rows;
  const uint32_t row = A.first_row + (valid ? r : A.rows - 1), V = A.vocab;
  const int32_t token = A.tokens[row];
  const T *x = static_cast<const T *>(A.x) + row_at(A.map, row).at[0];
  const bool mine = token >= 0 && gl < V;
  const float v = mine ? float(x[gl]) : -kInf;
  const uint32_t key = mine ? uint32_t(order_key(v, gl) >> 32) : 0;
  float m = lanes_max<L>(v, nullptr);
  const RowRef ref(A.c, m);
  const float z = m == -kInf ? -200.0f : fmaxf(ref.z(v), -200.0f), e = __builtin_amdgcn_exp2f(z);
  const float rest = lanes_sum<L>(v == m ? 0.0f : e, nullptr), ones = lanes_sum<L>(mine && v == m ? 1.0f : 0.0f, nullptr);
  const float s = lanes_sum<L>(e, nullptr), w = lanes_sum<L>(e * z, nullptr);
  uint32_t place = 0;
#pragma unroll
  for (int d = 1; d < L; ++d) {
    const uint32_t o = __shfl_xor(key, d);
    place += o > key || (o == key && (gl ^ d) < gl);
  }
  const float x_token = __shfl(v, token >= 0 && uint32_t(token) < V ? token : 0, L);
  const float l0 = log2_sum(rest, ones, ref.shift());
  if (!(fabsf(m) <= FLT_MAX) && m != -kInf) m = __builtin_nanf("");  // a NaN or an infinite logit
  if (!valid) return;
  if (gl == 0) {
    if (token < 0) pad_out(A, row);
    else row_out(A, row, token, x_token, m, s, w, ref.shift(), &l0);
  }
  if (mine && place < A.top) {
    const uint64_t at = uint64_t(row) * A.top + place;
    A.top_ids[at] = int32_t(gl);
    A.top_logp[at] = log_p(A, v, m, l0);
  }
  for (uint32_t k = (token < 0 ? 0 : V) + gl; k < A.top; k += L) put_top(A, row, k, 0, m, l0);
}

// The step over many long rows: a workgroup of 1024 lanes per CU that goes from row to row, the next one's units on
// their way into a second set of registers while this one is worked on. Rows are handed out as workgroups
// become free (in fixed turns the odd XCDs end some 8% after the even ones); a result does not depend on who works it
// out. [32768, 32000] in fp32: 1436 us, 5.84 TB/s, instead of 1585 with a workgroup per row (two of them fit a CU). With half
// the units, where more rows share a CU anyway, it loses: [32768, 8800] 522 us and 443, [32768, 16000] 743 and 709,
// [2048, 16000] 56 and 50; so do 16-bit rows, whose two exponentials a logit leave the memory idle at one workgroup per
// CU: 455 us and 425 at [16384, 32000] in bf16. Rows are whole units, 16-byte aligned in the gradient (the others'
// bounds cost registers that the two sets need).
constexpr uint32_t kStreamLanes = 1024, kStreamUnits = 8;
__device__ uint32_t g_stream_rows[2];  // rows handed out, workgroups that are done; zero between launches
__global__ __launch_bounds__(kStreamLanes) void held_stream_kernel(TokenArgs A) {
  typedef float T;
  constexpr uint32_t E = Unit<T>::E, L = kStreamLanes, N = kStreamUnits;
  __shared__ float lds[2][3][16];
  __shared__ uint32_t drawn[2];
  const uint32_t V = A.vocab, gl = threadIdx.x, grid = gridDim.x;
  typedef typename Unit<T>::vec vec;
  const auto fetch = [&](vec (&v)[N], uint32_t row, int32_t token) {
    const RowAt<2> at = row_at(A.map, row);
    const T *x = static_cast<const T *>(A.x) + at.at[0];
#pragma unroll
    for (uint32_t u = 0; u < N; ++u) {
      v[u] = T(-kInf);
      if (token >= 0 && (u * L + gl) * E < V) v[u] = load_unit(x + u * L * E + gl * E);
    }
  };
  uint32_t row = blockIdx.x, next = blockIdx.x + grid, turn = 0;
  int32_t token = A.tokens[row], next_token = next < A.rows ? A.tokens[next] : -1;
  vec first[N], second[N];
  fetch(first, row, token);
  // one row; the next one's loads are issued first
  const auto work = [&](vec (&v)[N], vec (&after)[N]) {
    uint32_t ticket = 0;  // an increment, not an add: its result is waited for where it is used, below
    if (gl == 0) ticket = atomicInc(&g_stream_rows[0], 0xffffffffu);
    if (next < A.rows) fetch(after, next, next_token);
    const RowAt<2> at = row_at(A.map, row);
    T *dx = static_cast<T *>(A.dx) + at.at[1];
    const float x_token = gl == 0 && uint32_t(token) < V ? float((static_cast<const T *>(A.x) + at.at[0])[token]) : 0.0f;
    float m = -kInf;
#pragma unroll
    for (uint32_t u = 0; u < N; ++u) m = __builtin_elementwise_maximum(m, unit_max(to_floats<T>(v[u])));
    if (gl == 0) drawn[turn] = ticket + 2 * grid;
    m = lanes_max<L>(m, lds[turn][0]);  // its barrier makes drawn[turn] visible too
    const uint32_t after_next = __builtin_amdgcn_readfirstlane(drawn[turn]);
    const int32_t after_token = after_next < A.rows ? A.tokens[after_next] : -1;
    // c (x - m) rather than a fused c x - c m: one more instruction, and no logits out of its range
    const auto exponent = [&](float x) { return fmaxf((x - m) * A.c, -200.0f); };
    float s = 0.0f, w = 0.0f;
#pragma unroll
    for (uint32_t u = 0; u < N; ++u) {
      const auto f = to_floats<T>(v[u]);
      auto terms = f;
#pragma unroll
      for (uint32_t e = 0; e < E; ++e) {
        const float z = exponent(f[e]);
        terms[e] = __builtin_amdgcn_exp2f(z);
        w = __builtin_fmaf(terms[e], z, w);
      }
      s += unit_sum(terms);
    }
    // both sums behind one barrier
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
      s += __shfl_xor(s, d);
      w += __shfl_xor(w, d);
    }
    if (gl % 64 == 0) {
      lds[turn][1][gl / 64] = s;
      lds[turn][2][gl / 64] = w;
    }
    __syncthreads();
    s = w = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < L / 64; ++k) {
      s += lds[turn][1][k];
      w += lds[turn][2][k];
    }
    if (!(fabsf(m) <= FLT_MAX) && m != -kInf) m = __builtin_nanf("");  // a NaN or an infinite logit
    const float l = log2f(s), h = kLn2 * (l - w / s);
    if (gl == 0) {
      if (token < 0) pad_out(A, row);
      else row_out(A, row, token, x_token, m, s, w, 0.0f);
    }
    RowGrad G(A, row, token, m, l, h < 0.0f ? 0.0f : h);
    if (m == -kInf) G.a = G.b = G.onehot = 0.0f;  // padding too
#pragma unroll
    for (uint32_t u = 0; u < N; ++u) {
      const uint32_t j = (u * L + gl) * E;
      if (j >= V) continue;
      auto f = to_floats<T>(v[u]);
#pragma unroll
      for (uint32_t e = 0; e < E; ++e) {
        const float z = exponent(f[e]);
        f[e] = -__builtin_amdgcn_exp2f(z) * __builtin_fmaf(G.b, z, G.a);
      }
      const uint32_t hit = uint32_t(token) - j;
      if (hit < E)
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) f[e] += hit == e ? G.onehot : 0.0f;
      __builtin_nontemporal_store(__builtin_convertvector(f, vec), reinterpret_cast<vec *>(dx + u * L * E + gl * E));
    }
    row = next, token = next_token;
    next = after_next, next_token = after_token;
    turn ^= 1;
  };
  while (row < A.rows) {
    work(first, second);
    if (row >= A.rows) break;
    work(second, first);
  }
  // the last workgroup leaves the counters at zero for the next launch
  if (gl == 0) {
    if (__hip_atomic_fetch_add(&g_stream_rows[1], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == grid - 1) {
      __hip_atomic_store(&g_stream_rows[0], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(&g_stream_rows[1], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
}

// f(lanes, units) for rows of `units` units that registers can hold; false for longer ones.
template <class F>
bool with_held_shape(uint32_t units, F &&f) {
  using std::integral_constant;
  const auto call = [&](auto l, auto n) { f(l, n); return true; };
#define HELD(l, n) \
  if (units <= l * n) return call(integral_constant<int, l>{}, integral_constant<int, n>{});
  HELD(2, 4) HELD(4, 4) HELD(8, 4) HELD(16, 4) HELD(32, 4) HELD(64, 4) HELD(256, 4) HELD(512, 4) HELD(1024, 4)
  HELD(1024, 8) HELD(1024, 16)
#undef HELD
  return false;
}

// ------------------------------------------------------------------------- host

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
  // the elements of a row, and of the units that its last workgroup has beyond it, stay within 31 bits
  if (V < 1 || V > (uint64_t(1) << 31) - 2 * kBwdUnits * kRowBlock * Unit<f16_t>::E) {
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
    if (overlapping(dx)) {
      report_error(where, "rows of x's gradient overlap");
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
    A.map.st[0][d] = s.st[0][d];
    A.map.st[1][d] = s.st[1][d];
  }
  return true;
}

// launch(args, workgroups) for parts of the rows that one grid of `threads` lanes holds.
template <class F>
void by_parts(const TokenArgs &A, uint64_t rows_per_block, uint64_t threads, F &&launch) {
  const uint64_t most = max_blocks(threads) * rows_per_block;
  TokenArgs part = A;
  for (uint64_t r = 0; r < A.rows; r += most) {
    part.first_row = uint32_t(r);
    part.rows = uint32_t(A.rows - r < most ? A.rows - r : most);
    launch(part, ceil_div(part.rows, rows_per_block));
  }
}

template <class T, int L, int U, bool GRAD>
void launch_held(const TokenArgs &A) {
  constexpr int B = L > kRowBlock ? L : kRowBlock;
  by_parts(A, L > 64 ? 1 : B / L, B, [](const TokenArgs &part, unsigned blocks) {
    held_kernel<T, L, U, GRAD><<<blocks, B, 0, stream()>>>(part);
  });
}

// Workgroups that a row is cut over: few rows, up to kCutBlocks workgroups of 1024 units or more.
uint32_t pieces_of(uint64_t rows, uint64_t vocab, uint64_t bytes) {
  uint64_t cut = vocab * bytes / 16 / 1024;
  if (cut > kCutBlocks / rows) cut = kCutBlocks / rows;
  return uint32_t(cut > kMaxPieces ? kMaxPieces : cut < 1 ? 1 : cut);
}
uint64_t pieces_bytes(uint64_t rows, uint64_t vocab, uint64_t bytes) {
  const uint32_t cut = pieces_of(rows, vocab, bytes);
  return cut > 1 ? rows * cut * sizeof(Piece) : 0;
}

// `room`: pieces_bytes of memory, or null to take them from the workspace.
template <class T, bool TOP>
bool launch_rows(const TokenArgs &A, void *room, const char *where) {
  const uint64_t unit = 16 / sizeof(T), units = A.vocab / unit;
  Pieces P{1, 1, 1, nullptr};
  if constexpr (!TOP)
    if (most_units<T>(A.vocab) <= 256) {
      with_held_shape(most_units<T>(A.vocab), [&](auto lanes, auto n) {
        constexpr int L = decltype(lanes)::value;
        if constexpr (L <= 64) launch_held<T, L, decltype(n)::value, false>(A);
      });
      return true;
    }
  if constexpr (TOP)
    if (A.vocab <= 64) {
      const auto tiny = [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        by_parts(A, kRowBlock / L, kRowBlock, [](const TokenArgs &part, unsigned blocks) {
          tiny_kernel<T, L><<<blocks, kRowBlock, 0, stream()>>>(part);
        });
      };
      if (A.vocab <= 16) tiny(std::integral_constant<int, 16>{});
      else if (A.vocab <= 32) tiny(std::integral_constant<int, 32>{});
      else tiny(std::integral_constant<int, 64>{});
      return true;
    }
  // A wave a row where rows are many and not long, four where a wave would be alone with its row for long: [4096,
  // 131072] in bf16 with 8 alternatives 224 us with one, 184 with four, [8192, 49999] in fp16 with 20 192 and 169;
  // [20000, 5000] in bf16 with 5 56 and 117. Rows of up to 640 units take one from half as many rows on: [4000, 2000] in fp32
  // with 5 14.3 and 17.7, [8000, 2600] with 20 36.3 and 40.1, but [1024, 2000] with 20 13.4 and 10.7, [4000, 4000] with 5 20.9
  // and 20.1. Rows of up to 256, one batch of a wave, always do.
  if (units <= 256 || (A.rows >= 4000 && units <= 640) || (A.rows >= 8192 && units < 4096)) {
    by_parts(A, 4, 256, [&](const TokenArgs &part, unsigned blocks) {
      fwd_kernel<T, 1, TOP, false><<<blocks, 256, 0, stream()>>>(part, P);
    });
    return true;
  }
  P.n = pieces_of(A.rows, A.vocab, sizeof(T));
  if (P.n > 1) {
    if (!room) room = partials(pieces_bytes(A.rows, A.vocab, sizeof(T)), where);
    P.found = static_cast<Piece *>(room);
    if (!P.found) return false;
    if constexpr (TOP) P.r = bound_key(A.top, P.n), P.q = ceil_div(A.top, P.r);
    fwd_kernel<T, 4, TOP, true><<<A.rows * P.n, 256, 0, stream()>>>(A, P);
  } else if (A.rows < 512 && units >= 6000) {
    // sixteen waves a row where a few hundred long ones leave the chip half empty: [300, 131072] in bf16 with 20
    // alternatives 40 us with sixteen, 57 with four, [300, 32000] in fp32 15.8 and 16.6; but [500, 32000] in bf16 13.4 and
    // 12.3, [500, 16000] with 5 16.0 and 13.1
    fwd_kernel<T, 16, TOP, false><<<A.rows, 1024, 0, stream()>>>(A, P);
  } else {
    by_parts(A, 1, 256, [&](const TokenArgs &part, unsigned blocks) {
      fwd_kernel<T, 4, TOP, false><<<blocks, 256, 0, stream()>>>(part, P);
    });
  }
  return true;
}

bool launch_forward(const TokenArgs &A, DTYPE type, void *room, const char *where) {
  bool ok = false;
  with_float_type(type, [&](auto t) {
    ok = A.top ? launch_rows<decltype(t), true>(A, room, where) : launch_rows<decltype(t), false>(A, room, where);
  });
  return ok;
}

// Whether every row of the gradient is whole 16-byte units at 16-byte addresses.
template <class T>
bool whole_rows(const TokenArgs &A) {
  constexpr int64_t E = Unit<T>::E;
  bool whole = A.vocab % E == 0 && aligned16(A.dx);
  for (int d = 0; d < A.map.rank; ++d) whole = whole && A.map.st[1][d] % E == 0;
  return whole;
}

// Units that a row of the gradient may lie in: one more than it fills where it is not `whole` units. The step over [32768,
// 1024] in fp32 72.7 us when whole rows are charged for one more too, 46.5 when not, [8192, 32768] 546 and 368, [32768, 2048]
// in bf16 95 and 49; forward and gradient of [32768, 2048] in fp32 180 and 133, of [32768, 4096] in bf16 179 and 132.
template <class T>
uint32_t grad_units(const TokenArgs &A, bool whole) {
  return whole ? A.vocab / Unit<T>::E : most_units<T>(A.vocab);
}

template <class T, bool ADD>
void launch_bwd(const TokenArgs &A) {
  const uint32_t units = grad_units<T>(A, whole_rows<T>(A));
  if (units < 128 && uint64_t(A.rows) * units < (uint64_t(1) << 32) - kRowBlock) {
    bwd_short_kernel<T, ADD><<<ceil_div(uint64_t(A.rows) * units, kRowBlock), kRowBlock, 0, stream()>>>(
        A, MagicDiv::make(units));
    return;
  }
  const uint32_t chunks = ceil_div(units, kBwdUnits * kRowBlock);
  const uint64_t most = max_blocks(kRowBlock) / chunks;  // rows of one launch
  TokenArgs part = A;
  for (uint64_t r = 0; r < A.rows; r += most) {
    part.first_row = uint32_t(r);
    part.rows = uint32_t(A.rows - r < most ? A.rows - r : most);
    bwd_kernel<T, ADD><<<part.rows * chunks, kRowBlock, 0, stream()>>>(part, chunks);
  }
}

void launch_backward(const TokenArgs &A, DTYPE type, bool add) {
  with_float_type(type, [&](auto t) {
    if (add) launch_bwd<decltype(t), true>(A);
    else launch_bwd<decltype(t), false>(A);
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
  if (!launch_forward(A, inputs[0]->dtype, nullptr, where)) return;
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
  bool held = false;
  with_float_type(x->dtype, [&](auto t) {
    typedef decltype(t) T;
    const bool whole = whole_rows<T>(A);
    const uint32_t in_row = grad_units<T>(A, whole);
    // Sixteen units a lane spill some 25 registers, and take a workgroup per row: they pay in fp32 where rows fill the
    // chip ([8192, 65000] 965 us and 1058 in two passes, [400, 65000] 58 and 67; but [64, 65000] 21.6 and 20.3, [4, 65000]
    // 17.8 and 12.9), not in 16 bits, where a lane has twice the logits ([8192, 65600] in bf16 699 and 503, [8192, 131000]
    // 1109 and 1069, [4, 131000] 27 and 13).
    const uint32_t most = sizeof(T) == 4 && A.rows >= uint32_t(num_cus()) ? 16 * 1024 : 8 * 1024;
    held = in_row <= most && with_held_shape(in_row, [&](auto lanes, auto units) {
      constexpr int L = decltype(lanes)::value;
      constexpr int U = decltype(units)::value;
      if constexpr (L == kStreamLanes && U == kStreamUnits && sizeof(T) == 4) {
        if (A.rows >= 4 * uint32_t(num_cus()) && whole) {
          held_stream_kernel<<<num_cus(), kStreamLanes, 0, stream()>>>(A);
          return;
        }
      }
      if constexpr (U < 16 || sizeof(T) == 4) launch_held<T, L, U, true>(A);
    });
  });
  if (held) {
    finish(where);
    return;
  }
  // the statistics between the two, and the pieces of cut rows after them
  const uint64_t stats = (2 * N * sizeof(float) + 255) / 256 * 256;
  char *work = static_cast<char *>(partials(stats + pieces_bytes(N, A.vocab, float_bytes(x)), where));
  if (!work) return;
  A.stats = reinterpret_cast<float *>(work);
  if (!launch_forward(A, x->dtype, work + stats, where)) return;
  launch_backward(A, x->dtype, false);
  finish(where);
}

}  // extern "C"
