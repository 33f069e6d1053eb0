// places.hpp — whether two strided operands share memory: host code without HIP, so that the CPU tests compare it with a
// count of bytes over small operands.
#pragma once

#include <cstdint>

#include "plast_abi.h"

namespace plast {

inline int element_bytes(const Tensor *t) { return t->dtype == INT64 ? 8 : t->dtype == FLOAT16 || t->dtype == BFLOAT16 ? 2 : 4; }

// The bytes of a tensor: runs of `run` bytes, at `at` and any of the multiples below n[d] of step[d] from there, the axes
// by falling steps. Axes whose steps leave no gap are part of the run.
struct Place {
  typedef __int128 wide;  // no product of the strides and extents that a tensor can name leaves it
  wide at = 0, run = 0;   // run 0: no bytes
  int rank = 0;
  wide n[PLAST_MAX_NDIM], step[PLAST_MAX_NDIM];

  Place() = default;
  explicit Place(const Tensor *t) {
    if (!t || !t->data || t->ndim > PLAST_MAX_NDIM) return;
    const int bytes = element_bytes(t);
    at = wide(reinterpret_cast<uintptr_t>(t->data));
    wide ext[PLAST_MAX_NDIM], st[PLAST_MAX_NDIM];
    int axes = 0;
    for (uint64_t d = 0; d < t->ndim; ++d) {
      if (t->shape[d] == 0) return;
      wide s = wide(int64_t(t->strides[d])) * bytes;
      if (t->shape[d] == 1 || s == 0) continue;
      if (s < 0) {
        at += s * wide(t->shape[d] - 1);
        s = -s;
      }
      int i = axes++;  // by rising steps
      for (; i > 0 && st[i - 1] > s; --i) ext[i] = ext[i - 1], st[i] = st[i - 1];
      ext[i] = wide(t->shape[d]), st[i] = s;
    }
    run = bytes;
    int i = 0;
    for (; i < axes && st[i] <= run; ++i) run += st[i] * (ext[i] - 1);
    rank = axes - i;
    for (int d = 0; d < rank; ++d) n[d] = ext[axes - 1 - d], step[d] = st[axes - 1 - d];
  }
  wide span(int from = 0) const {
    wide s = run;
    for (int d = from; d < rank; ++d) s += step[d] * (n[d] - 1);
    return s;
  }
};

namespace places {

inline Place::wide floor_div(Place::wide a, Place::wide b) { return a / b - (a % b < 0); }  // b > 0

// Whether a, from axis i on and starting at `pa`, and b, from axis j on and starting at `pb`, share a byte. Each pair of parts
// looked at takes one of `looks`; with none left they count as sharing.
inline bool meet(const Place &a, int i, Place::wide pa, const Place &b, int j, Place::wide pb, int &looks) {
  typedef Place::wide wide;
  if (pa >= pb + b.span(j) || pb >= pa + a.span(i)) return false;
  if ((i == a.rank && j == b.rank) || --looks < 0) return true;
  if (i == a.rank || (j < b.rank && b.step[j] > a.step[i])) return meet(b, j, pb, a, i, pa, looks);
  // the parts of a along its axis i, `inner` bytes each; along an axis that b steps through as far, only the difference counts
  const bool both = j < b.rank && b.step[j] == a.step[i];
  const wide s = a.step[i], inner = a.span(i + 1), other = b.span(both ? j + 1 : j);
  wide lo = floor_div(pb - pa - inner, s) + 1, hi = floor_div(pb - pa + other - 1, s);
  const wide least = both ? 1 - b.n[j] : 0, most = a.n[i] - 1;
  if (lo < least) lo = least;
  if (hi > most) hi = most;
  for (wide k = lo; k <= hi; ++k)
    if (meet(a, i + 1, pa + k * s, b, both ? j + 1 : j, pb, looks)) return true;
  return false;
}

}  // namespace places

// Whether a and b share a byte. Operands of one layout in one buffer (halves of a projection, say) are told apart in a few steps;
// layouts that interleave with other steps and are not told apart in kLooks count as sharing.
constexpr int kLooks = 1 << 14;
inline bool share_memory(const Place &a, const Place &b) {
  if (a.run == 0 || b.run == 0) return false;
  int looks = kLooks;
  return places::meet(a, 0, a.at, b, 0, b.at, looks);
}

// The first byte of a tensor and the one behind its last, what tells most operands apart; all of memory where 64 bits do not hold
// them. Of seven operands and their pairs they take 0.1 us of a call, Places 0.5.
struct Span {
  int64_t lo = 0, hi = 0;  // equal: no bytes
  explicit Span(const Tensor *t) {
    if (!t || !t->data || t->ndim > PLAST_MAX_NDIM) return;
    const int64_t bytes = element_bytes(t);
    int64_t below = 0, above = 1;
    bool over = false;
    for (uint64_t d = 0; d < t->ndim; ++d) {
      if (t->shape[d] == 0) return;
      int64_t s;
      over |= __builtin_mul_overflow(int64_t(t->strides[d]), t->shape[d] - 1, &s);
      over |= s < 0 ? __builtin_add_overflow(below, s, &below) : __builtin_add_overflow(above, s, &above);
    }
    const int64_t at = int64_t(reinterpret_cast<uintptr_t>(t->data));
    over |= __builtin_mul_overflow(below, bytes, &below);
    over |= __builtin_mul_overflow(above, bytes, &above);
    over |= __builtin_add_overflow(at, below, &lo);
    over |= __builtin_add_overflow(at, above, &hi);
    if (over) lo = INT64_MIN, hi = INT64_MAX;
  }
  bool meets(const Span &o) const { return lo < o.hi && o.lo < hi && lo < hi && o.lo < o.hi; }
};

}  // namespace plast
