// clip.hip — the global norm of the gradients of a list of parameters, and their scaling to a bound on it:
//   norm = sqrt(sum over all elements of all gradients of g^2);  where norm > bound: g = g bound / norm.
// Squares are summed and gradients scaled in 64 bits, and rounded to fp32 and from there to their type: no gradient's square,
// and no factor, leaves their range, and the sum has fp32's digits whatever its order (a conversion and a multiply-add an
// element, far below the read's time).
//
// Two launches: the first one's workgroups take equal runs of the gradients' pieces and leave a sum each; those of the second
// add all sums up, each for itself and in one order, and scale. A small set is bound by the two launches (four gradients of
// 0.5 MB in all 9.4 us); others by the read (1.07 GB within the bound 160 us, 6.7 TB/s) and, past the bound, by reading again
// and writing (24 gradients of 1024 x 1024: 21 us, then 35, 5.7 TB/s).
#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <type_traits>
#include <vector>

#include "rows.hpp"

namespace plast {
namespace {

constexpr int kGroup = 160;     // gradients whose table fits a kernel's arguments
constexpr int kLanes = 256;
constexpr uint32_t kUnits = 4;  // of 16 bytes, of a lane in a piece
constexpr uint64_t kPiece = uint64_t(kLanes) * kUnits * 16;  // bytes
constexpr uint64_t kCached = uint64_t(256) << 20;  // bytes of the last-level cache
// A launch's workgroups: up to kFewPieces pieces have one each in either launch, so that each XCD scales what its
// own cache has read ([4, 1024, 1024] in fp32 15 us, 21 otherwise). More are summed by kSumBlocks in one run each (1.07 GB 163 us,
// 6.6 TB/s; 172 with 2048) and scaled by kScaleBlocks in turns of kRun (150 gradients of 1.2 MB 135 us, 172 piece by piece, whose
// table is looked up for each; one run each 148; 1.07 GB 593, 558 and 685 in all).
constexpr uint32_t kFewPieces = 2048, kSumBlocks = 1024, kScaleBlocks = 2048, kRun = 2;

struct Entry {
  char *p;
  uint64_t n;            // elements
  uint32_t first, type;  // first: the number of its first piece
};
// Gradients, in the kernel's arguments or in device memory. of(): the one that piece p is of, the last whose first piece is at or
// before it.
struct InArguments {
  Entry e[kGroup];
  __device__ __forceinline__ const Entry &operator[](int i) const { return e[i]; }
  __device__ __forceinline__ int of(int count, uint32_t p) const {
    int i = 0, hi = count - 1;
    while (i < hi) {
      const int mid = (i + hi + 1) >> 1;
      if (e[mid].first <= p) i = mid;
      else hi = mid - 1;
    }
    return i;
  }
};
struct InMemory {
  const Entry *e;
  __device__ __forceinline__ const Entry &operator[](int i) const { return e[i]; }
  // by a wave, 64 at a time: two looks for up to 4096 gradients
  __device__ __forceinline__ int of(int count, uint32_t p) const {
    int at = 0, span = count;
    while (span > 1) {
      const int step = (span + 63) / 64, i = int(threadIdx.x & 63) * step;
      const bool before = i < span && e[at + (i < span ? i : 0)].first <= p;
      const int last = (__popcll(__ballot(before)) - 1) * step;
      at += last;
      span = span - last < step ? span - last : step;
    }
    return __builtin_amdgcn_readfirstlane(at);
  }
};
// f(entry, first, end) for the pieces [first, end) of the table's that each entry has, pieces of the entry.
template <class Table, class F>
__device__ __forceinline__ void for_entries(const Table &T, int count, uint32_t first, uint32_t end, F &&f) {
  if (first >= end) return;
  for (int i = T.of(count, first); i < count; ++i) {
    const Entry E = T[i];
    const uint32_t behind = i + 1 < count ? T[i + 1].first : 0xffffffffu;
    const uint32_t p0 = E.first > first ? E.first : first, p1 = behind < end ? behind : end;
    f(E, p0 - E.first, p1 - E.first);
    if (behind >= end) return;
  }
}

struct ClipRun {
  int count;
  uint32_t pieces, per, run;  // per: of a workgroup that sums; run: of one that scales, in each of its turns
};

__device__ __forceinline__ double block_sum(double s, double *lds) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  s = lds[0];
#pragma unroll
  for (int w = 1; w < kLanes / 64; ++w) s += lds[w];
  return s;
}

template <class T>
constexpr uint32_t kPieceOf = kPiece / sizeof(T);  // elements

// A lane's units of a whole piece.
template <class T, bool NT>
struct Units {
  typename Unit<T>::vec v[kUnits];
  __device__ __forceinline__ void load(const T *g, uint32_t piece) {
    const T *p = g + uint64_t(piece) * kPieceOf<T> + threadIdx.x * Unit<T>::E;
#pragma unroll
    for (uint32_t u = 0; u < kUnits; ++u) {
      const auto *q = reinterpret_cast<const typename Unit<T>::any *>(p + u * kLanes * Unit<T>::E);
      if constexpr (NT) v[u] = __builtin_nontemporal_load(q);
      else v[u] = *q;
    }
  }
};
// f(element) for a lane's elements of a last piece, which is not whole.
template <class T, class F>
__device__ __forceinline__ void for_rest(T *g, uint64_t n, uint32_t piece, F &&f) {
  for (uint64_t j = uint64_t(piece) * kPieceOf<T> + threadIdx.x; j < n; j += kLanes) f(g[j]);
}

// The sum of the squares of pieces [p, end) of a gradient: the next piece's units on their way, a sum for each unit.
template <class T, bool NT>
__device__ __forceinline__ double squares(const Entry &E, uint32_t p, uint32_t end) {
  const T *g = reinterpret_cast<const T *>(E.p);
  const uint32_t whole = uint32_t(E.n / kPieceOf<T>), stop = end < whole ? end : whole;
  double s[kUnits] = {};
  if (p < stop) {
    Units<T, NT> now, next;
    now.load(g, p);
    for (;;) {
      const bool more = ++p < stop;
      if (more) next.load(g, p);
#pragma unroll
      for (uint32_t u = 0; u < kUnits; ++u) {
        const typename Unit<T>::floats f = to_floats<T>(now.v[u]);
#pragma unroll
        for (uint32_t e = 0; e < Unit<T>::E; ++e) s[u] = __builtin_fma(double(f[e]), double(f[e]), s[u]);
      }
      if (!more) break;
      now = next;
    }
  }
  if (end > whole)
    for_rest(const_cast<T *>(g), E.n, whole, [&](T &v) {
      const double f = double(float(v));
      s[0] = __builtin_fma(f, f, s[0]);
    });
  return (s[0] + s[1]) + (s[2] + s[3]);
}
static_assert(kUnits == 4, "four sums");

// Pieces [p, end) times scale, the next one's units on their way.
template <class T>
__device__ __forceinline__ void scale_pieces(const Entry &E, uint32_t p, uint32_t end, double scale) {
  T *g = reinterpret_cast<T *>(E.p);
  const uint32_t whole = uint32_t(E.n / kPieceOf<T>), stop = end < whole ? end : whole;
  if (p < stop) {
    Units<T, false> now, next;
    now.load(g, p);
    for (;;) {
      T *to = g + uint64_t(p) * kPieceOf<T> + threadIdx.x * Unit<T>::E;
      const bool more = ++p < stop;
      if (more) next.load(g, p);
#pragma unroll
      for (uint32_t u = 0; u < kUnits; ++u) {
        typename Unit<T>::floats f = to_floats<T>(now.v[u]);
#pragma unroll
        for (uint32_t e = 0; e < Unit<T>::E; ++e) f[e] = float(double(f[e]) * scale);
        __builtin_nontemporal_store(__builtin_convertvector(f, typename Unit<T>::vec),
                                    reinterpret_cast<typename Unit<T>::any *>(to + u * kLanes * Unit<T>::E));
      }
      if (!more) break;
      now = next;
    }
  }
  if (end > whole) for_rest(g, E.n, whole, [&](T &v) { v = T(float(double(float(v)) * scale)); });
}

template <class Table, bool NT>
__global__ __launch_bounds__(kLanes) void squares_kernel(Table A, ClipRun R, double *sums) {
  __shared__ double lds[kLanes / 64];
  const uint32_t first = blockIdx.x * R.per, end = first + R.per < R.pieces ? first + R.per : R.pieces;
  double s = 0.0;
  for_entries(A, R.count, first, end, [&](const Entry &E, uint32_t p, uint32_t to) {
    if (E.type == FLOAT32) s += squares<float, NT>(E, p, to);
    else if (E.type == FLOAT16) s += squares<f16_t, NT>(E, p, to);
    else s += squares<bf16_t, NT>(E, p, to);
  });
  s = block_sum(s, lds);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

template <class Table>
__global__ __launch_bounds__(kLanes) void scale_kernel(Table A, ClipRun R, const double *sums, uint32_t n, float bound,
                                                       float *norm_out) {
  __shared__ double lds[kLanes / 64];
  double s = 0.0;
#pragma unroll 8
  for (uint32_t i = threadIdx.x; i < n; i += kLanes) s += sums[i];
  const double norm = sqrt(block_sum(s, lds));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = float(norm);
  if (!(norm > double(bound)) || norm == __builtin_huge_val()) return;  // within the bound, or not finite
  const double scale = double(bound) / norm;
  for (uint64_t p = uint64_t(blockIdx.x) * R.run; p < R.pieces; p += uint64_t(gridDim.x) * R.run) {
    const uint32_t first = uint32_t(p), end = R.pieces - first < R.run ? R.pieces : first + R.run;
    for_entries(A, R.count, first, end, [&](const Entry &E, uint32_t q, uint32_t to) {
      if (E.type == FLOAT32) scale_pieces<float>(E, q, to, scale);
      else if (E.type == FLOAT16) scale_pieces<f16_t>(E, q, to, scale);
      else scale_pieces<bf16_t>(E, q, to, scale);
    });
  }
}

// Part of a longer table to device memory, from the arguments: a copy from the host would have to keep its source until it is done, or be
// waited for. us, this / a table copied and kept for as long as the calls' gradients are the same: 400 gradients of 3 KB 20 / 11, of
// other addresses in each call 21 / 31; 400 of 0.8 MB 161 / 155 and 209 / 226.
__global__ __launch_bounds__(kLanes) void table_kernel(InArguments A, int count, Entry *to) {
  if (int(threadIdx.x) < count) to[threadIdx.x] = A.e[threadIdx.x];
}
static_assert(kGroup <= kLanes, "a lane an entry");

// ------------------------------------------------------------------------- host

const char *const where = "clip_grad_norm_hip";

// Whether two of the gradients share memory: one scaled by two workgroups at once would be scaled twice, or once.
bool share_memory(std::vector<std::pair<uint64_t, uint64_t>> &spans) {
  const auto meet = [&]() {
    for (size_t i = 1; i < spans.size(); ++i)
      if (spans[i].first < spans[i - 1].second) return true;
    return false;
  };
  if (!meet()) return false;  // in the order of their addresses already, most often
  std::sort(spans.begin(), spans.end());
  return meet();
}

}  // namespace
}  // namespace plast

using namespace plast;

extern "C" {

void clip_grad_norm_hip(Tensor **parameters, int num_parameters, float max_norm, Tensor *norm) try {
  if (!(max_norm >= 0.0f)) {
    report_error(where, "max_norm must be at least 0, not %g", double(max_norm));
    return;
  }
  if (norm && !f32_vector(norm, 1)) {
    report_error(where, "norm must be a FLOAT32 GPU tensor of one element");
    return;
  }
  std::vector<Entry> entries;
  std::vector<std::pair<uint64_t, uint64_t>> spans;
  uint64_t pieces = 0;
  if (parameters && num_parameters > 0) entries.reserve(size_t(num_parameters)), spans.reserve(size_t(num_parameters));
  for (int k = 0; parameters && k < num_parameters; ++k) {
    const Tensor *t = parameters[k];
    if (!t || !t->grad) continue;
    const Tensor *g = t->grad;
    const uint64_t n = numel(g);
    if (n == 0) continue;
    if (g->device != GPU || !is_float(g) || !contiguous(g) || !g->data || n != numel(t)) {
      report_error(where, "the gradient of parameter %d is not a contiguous GPU tensor of FLOAT32, FLOAT16 or BFLOAT16 of its "
                   "size", k);
      return;
    }
    const uint64_t bytes = n * float_bytes(g), at = reinterpret_cast<uint64_t>(g->data);
    entries.push_back({static_cast<char *>(g->data), n, uint32_t(pieces), uint32_t(g->dtype)});
    pieces += (bytes + kPiece - 1) / kPiece;
    spans.emplace_back(at, at + bytes);
  }
  if (pieces >= uint64_t(1) << 32) {
    report_error(where, "gradients of more than 2^46 bytes");
    return;
  }
  if (norm) spans.emplace_back(reinterpret_cast<uint64_t>(norm->data), reinterpret_cast<uint64_t>(norm->data) + sizeof(float));
  if (share_memory(spans)) {
    report_error(where, "two gradients, or the norm and one of them, share memory, or a parameter is listed twice");
    return;
  }
  if ((entries.empty() && !norm) || !ensure_init()) return;

  const uint32_t n = uint32_t(pieces), per = n <= kFewPieces ? 1 : ceil_div(n, kSumBlocks), sums = n ? ceil_div(n, per) : 1;
  const uint32_t run = n <= kFewPieces ? 1 : kRun, blocks = n <= kFewPieces ? sums : std::min(ceil_div(n, run), kScaleBlocks);
  const bool many = entries.size() > size_t(kGroup);
  char *room = static_cast<char *>(partials(sums * sizeof(double) + (many ? entries.size() * sizeof(Entry) : 0), where));
  if (!room) return;
  double *const to = reinterpret_cast<double *>(room);
  float *const out = norm ? static_cast<float *>(norm->data) : nullptr;
  const ClipRun R{int(entries.size()), n, per, run};
  const auto launch = [&](const auto &table) {
    typedef std::decay_t<decltype(table)> Table;
    if (pieces * kPiece > kCached) squares_kernel<Table, true><<<sums, kLanes, 0, stream()>>>(table, R, to);
    else squares_kernel<Table, false><<<sums, kLanes, 0, stream()>>>(table, R, to);
    scale_kernel<Table><<<blocks, kLanes, 0, stream()>>>(table, R, to, sums, max_norm, out);
  };
  InArguments A;
  memset(&A, 0, sizeof A);
  if (!many) {
    std::copy(entries.begin(), entries.end(), A.e);
    launch(A);
  } else {
    Entry *const table = reinterpret_cast<Entry *>(to + sums);
    for (size_t i = 0; i < entries.size(); i += kGroup) {
      const size_t m = std::min(entries.size() - i, size_t(kGroup));
      std::copy_n(entries.begin() + i, m, A.e);
      table_kernel<<<1, kLanes, 0, stream()>>>(A, int(m), table + i);
    }
    launch(InMemory{table});
  }
  finish(where);
} catch (const std::bad_alloc &) {
  report_error(where, "no host memory for the tables of %d gradients", num_parameters);
}

}  // extern "C"
