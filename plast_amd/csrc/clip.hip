// clip.hip — the global norm of the gradients of a list of parameters, and their scaling to a bound on it:
//   norm = sqrt(sum over all elements of all gradients of g^2);  where norm > bound: g = g bound / norm.
// Squares are summed and gradients scaled in 64 bits: no gradient's square, and no factor, leaves their range, and the sum
// has fp32's digits whatever its order (a conversion and a multiply-add an element, far below the read's time).
//
// Two launches: a launch's workgroups take equal runs of the gradients' pieces and leave a sum each; those of the second add
// all sums up, each for itself and in one order, and scale the pieces they had, the last read first.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>
#include <vector>

#include "opt_plan.hpp"
#include "rows.hpp"

namespace plast {
namespace {

constexpr int kGroup = 96;      // tensors of a launch whose table is in the kernel's arguments
constexpr int kLanes = 256;
constexpr uint32_t kUnits = 4;  // of 16 bytes, of a lane in a piece
constexpr uint64_t kPiece = uint64_t(kLanes) * kUnits * 16;  // bytes
constexpr uint32_t kMostBlocks = 2048;  // of all launches together, eight to a CU

// A gradient: p, n, the number of its first piece; its type in vec.
struct ClipTable {
  OptEntry e[kGroup];
};

// f(entry, piece of the entry) for pieces [first, end) of the table's, in order or from the last.
template <bool BACK, class F>
__device__ __forceinline__ void for_pieces(const OptEntry *T, int count, uint32_t first, uint32_t end, F &&f) {
  if (first >= end) return;
  const uint32_t at = BACK ? end - 1 : first;
  int i = 0, hi = count - 1;
  while (i < hi) {
    const int mid = (i + hi + 1) >> 1;
    if (T[mid].first_block <= at) i = mid;
    else hi = mid - 1;
  }
  if (BACK) {
    for (uint32_t p = end; p-- > first;) {
      while (T[i].first_block > p) --i;
      f(T[i], p - T[i].first_block);
    }
  } else {
    for (uint32_t p = first; p < end; ++p) {
      while (i + 1 < count && T[i + 1].first_block <= p) ++i;
      f(T[i], p - T[i].first_block);
    }
  }
}

// Every launch's share of the work.
struct ClipRun {
  const OptEntry *table;  // null: in the arguments
  int count;
  uint32_t pieces, per;   // per: of a workgroup
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
__device__ __forceinline__ double piece_squares(const OptEntry &E, uint32_t piece) {
  constexpr uint32_t W = Unit<T>::E;
  const T *g = reinterpret_cast<const T *>(E.p);
  const uint64_t at = uint64_t(piece) * (kPiece / sizeof(T)) + threadIdx.x * W;
  double s = 0.0;
  if (uint64_t(piece + 1) * (kPiece / sizeof(T)) <= E.n) {
    typename Unit<T>::vec v[kUnits];
#pragma unroll
    for (uint32_t u = 0; u < kUnits; ++u) v[u] = *reinterpret_cast<const typename Unit<T>::any *>(g + at + u * kLanes * W);
#pragma unroll
    for (uint32_t u = 0; u < kUnits; ++u) {
      const typename Unit<T>::floats f = to_floats<T>(v[u]);
#pragma unroll
      for (uint32_t e = 0; e < W; ++e) s = __builtin_fma(double(f[e]), double(f[e]), s);
    }
    return s;
  }
  for (uint32_t u = 0; u < kUnits; ++u)
    for (uint32_t e = 0; e < W; ++e) {
      const uint64_t j = at + u * kLanes * W + e;
      if (j < E.n) {
        const double f = double(float(g[j]));
        s = __builtin_fma(f, f, s);
      }
    }
  return s;
}

template <class T>
__device__ __forceinline__ void scale_piece(const OptEntry &E, uint32_t piece, double scale) {
  constexpr uint32_t W = Unit<T>::E;
  T *g = reinterpret_cast<T *>(E.p);
  const uint64_t at = uint64_t(piece) * (kPiece / sizeof(T)) + threadIdx.x * W;
  if (uint64_t(piece + 1) * (kPiece / sizeof(T)) <= E.n) {
    typename Unit<T>::vec v[kUnits];
#pragma unroll
    for (uint32_t u = 0; u < kUnits; ++u) v[u] = *reinterpret_cast<const typename Unit<T>::any *>(g + at + u * kLanes * W);
#pragma unroll
    for (uint32_t u = 0; u < kUnits; ++u) {
      typename Unit<T>::floats f = to_floats<T>(v[u]);
#pragma unroll
      for (uint32_t e = 0; e < W; ++e) f[e] = float(double(f[e]) * scale);
      *reinterpret_cast<typename Unit<T>::any *>(g + at + u * kLanes * W) =
          __builtin_convertvector(f, typename Unit<T>::vec);
    }
    return;
  }
  for (uint32_t u = 0; u < kUnits; ++u)
    for (uint32_t e = 0; e < W; ++e) {
      const uint64_t j = at + u * kLanes * W + e;
      if (j < E.n) g[j] = T(float(double(float(g[j])) * scale));
    }
}

__global__ __launch_bounds__(kLanes) void squares_kernel(ClipTable A, ClipRun R, double *sums) {
  __shared__ double lds[kLanes / 64];
  const uint32_t first = blockIdx.x * R.per, end = first + R.per < R.pieces ? first + R.per : R.pieces;
  double s = 0.0;
  for_pieces<false>(R.table ? R.table : A.e, R.count, first, end, [&](const OptEntry &E, uint32_t piece) {
    if (E.vec == FLOAT32) s += piece_squares<float>(E, piece);
    else if (E.vec == FLOAT16) s += piece_squares<f16_t>(E, piece);
    else s += piece_squares<bf16_t>(E, piece);
  });
  s = block_sum(s, lds);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

__global__ __launch_bounds__(kLanes) void scale_kernel(ClipTable A, ClipRun R, const double *sums, uint32_t n, float bound,
                                                       float *norm_out) {
  __shared__ double lds[kLanes / 64];
  double s = 0.0;
  for (uint32_t i = threadIdx.x; i < n; i += kLanes) s += sums[i];
  const double norm = sqrt(block_sum(s, lds));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = float(norm);
  if (!(norm > double(bound)) || norm == __builtin_huge_val()) return;  // within the bound, or not finite
  const double scale = double(bound) / norm;
  const uint32_t first = blockIdx.x * R.per, end = first + R.per < R.pieces ? first + R.per : R.pieces;
  for_pieces<true>(R.table ? R.table : A.e, R.count, first, end, [&](const OptEntry &E, uint32_t piece) {
    if (E.vec == FLOAT32) scale_piece<float>(E, piece, scale);
    else if (E.vec == FLOAT16) scale_piece<f16_t>(E, piece, scale);
    else scale_piece<bf16_t>(E, piece, scale);
  });
}

// ------------------------------------------------------------------------- host

std::mutex g_table_mu;
OptTableCache g_table;  // of the last call with more than kGroup gradients

const OptEntry *device_table(const std::vector<OptEntry> &e, const char *where) {
  return g_table.get(
      e,
      [&]() {
        if (hipStreamSynchronize(stream()) == hipSuccess) return true;
        report_error(where, "waiting for the library stream failed");
        return false;
      },
      [&](size_t n) -> OptEntry * {
        OptEntry *p = nullptr;
        if (hipMalloc(&p, n * sizeof(OptEntry)) == hipSuccess) return p;
        report_error(where, "allocation of the tensor table (%zu entries) failed", n);
        return nullptr;
      },
      [](OptEntry *p) { (void)hipFree(p); },
      [&](OptEntry *dst, const std::vector<OptEntry> &src) {
        if (hipMemcpyAsync(dst, src.data(), src.size() * sizeof(OptEntry), hipMemcpyHostToDevice, stream()) == hipSuccess &&
            hipStreamSynchronize(stream()) == hipSuccess)
          return true;
        report_error(where, "upload of the tensor table failed");
        return false;
      });
}

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

void clip_grad_norm_hip(Tensor **parameters, int num_parameters, float max_norm, Tensor *norm) {
  const char *where = "clip_grad_norm_hip";
  if (!(max_norm >= 0.0f)) {
    report_error(where, "max_norm must be at least 0, not %g", double(max_norm));
    return;
  }
  if (norm && !f32_vector(norm, 1)) {
    report_error(where, "norm must be a FLOAT32 GPU tensor of one element");
    return;
  }
  std::vector<OptEntry> entries;
  std::vector<std::pair<uint64_t, uint64_t>> spans;
  uint64_t pieces = 0;
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
    OptEntry e;
    memset(&e, 0, sizeof e);
    e.p = static_cast<float *>(g->data);
    e.n = n;
    e.first_block = uint32_t(pieces);
    e.vec = uint32_t(g->dtype);
    const uint64_t bytes = n * float_bytes(g), at = reinterpret_cast<uint64_t>(g->data);
    pieces += (bytes + kPiece - 1) / kPiece;
    entries.push_back(e);
    spans.emplace_back(at, at + bytes);
  }
  if (pieces >= uint64_t(1) << 32) {
    report_error(where, "gradients of more than 2^46 bytes");
    return;
  }
  if (share_memory(spans)) {
    report_error(where, "two gradients share memory, or a parameter is listed twice");
    return;
  }
  if ((entries.empty() && !norm) || !ensure_init()) return;

  // the launches: one over a table in device memory, or, in a capture, one for each kGroup gradients
  const bool table = entries.size() > size_t(kGroup) && !capturing();
  const size_t group = table ? entries.size() : size_t(kGroup);
  const size_t launches = entries.empty() ? 1 : (entries.size() + group - 1) / group;
  const uint32_t most = uint32_t(std::max<size_t>(1, kMostBlocks / launches));
  std::lock_guard<std::mutex> lk(g_table_mu);
  const OptEntry *T = table ? device_table(entries, where) : nullptr;
  if (table && !T) return;
  struct Launch {
    ClipRun run;
    uint32_t blocks, first_sum;
  };
  std::vector<Launch> plan;
  uint32_t sums = 0;
  for (size_t i = 0; i < launches; ++i) {
    const size_t a = i * group, b = std::min(entries.size(), a + group);
    const uint64_t p0 = a < b ? entries[a].first_block : 0, p1 = b < entries.size() ? entries[b].first_block : pieces;
    const uint32_t n = uint32_t(p1 - p0), per = n ? ceil_div(n, most) : 1, blocks = n ? ceil_div(n, per) : 1;
    plan.push_back({{T, int(b - a), n, per}, blocks, sums});
    sums += blocks;
  }
  double *room = static_cast<double *>(partials(sums * sizeof(double), where));
  if (!room) return;
  const auto arguments = [&](size_t i) {
    ClipTable A;
    memset(&A, 0, sizeof A);
    if (!T)
      for (int k = 0; k < plan[i].run.count; ++k) {
        A.e[k] = entries[i * group + k];
        A.e[k].first_block -= entries[i * group].first_block;
      }
    return A;
  };
  for (size_t i = 0; i < launches; ++i)
    squares_kernel<<<plan[i].blocks, kLanes, 0, stream()>>>(arguments(i), plan[i].run, room + plan[i].first_sum);
  for (size_t i = 0; i < launches; ++i)
    scale_kernel<<<plan[i].blocks, kLanes, 0, stream()>>>(arguments(i), plan[i].run, room, sums, max_norm,
                                                          i == 0 && norm ? static_cast<float *>(norm->data) : nullptr);
  finish(where);
}

}  // extern "C"
