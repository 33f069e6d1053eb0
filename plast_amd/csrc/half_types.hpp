// half_types.hpp — the element types of the operators that take 16-bit floats beside fp32: device
// types by DTYPE, a dispatch over them, and the check of strides that are written through.
#pragma once

#include "common.hpp"

namespace plast {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

inline bool is_float(const Tensor *t) { return t->dtype == FLOAT32 || is_half(t); }
inline uint64_t float_bytes(const Tensor *t) { return is_half(t) ? 2 : 4; }

// f(T{}) with T the device type of a float dtype.
template <class F>
void with_float_type(DTYPE d, F &&f) {
  if (d == FLOAT16) f(f16_t{});
  else if (d == BFLOAT16) f(bf16_t{});
  else f(float{});
}

// Whether elements of t can lie at one address: an axis of several elements, in order of their strides, does not step
// past what the ones below it span (every second column of rows of 7 does: strides 7 and 2).
inline bool overlapping(const Tensor *t) {
  const auto step = [&](uint64_t d) {
    const int64_t s = int64_t(t->strides[d]);
    return s < 0 ? -uint64_t(s) : uint64_t(s);
  };
  uint64_t span = 0;
  bool done[PLAST_MAX_NDIM] = {};
  for (uint64_t k = 0; k < t->ndim; ++k) {
    uint64_t at = t->ndim;
    for (uint64_t d = 0; d < t->ndim; ++d)
      if (!done[d] && (at == t->ndim || step(d) < step(at))) at = d;
    done[at] = true;
    if (t->shape[at] <= 1) continue;
    if (step(at) <= span) return true;
    span += step(at) * (t->shape[at] - 1);
  }
  return false;
}

}  // namespace plast
