// half_types.hpp — the element types of the operators that take 16-bit floats beside fp32: device
// types by DTYPE, and a dispatch over them.
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

}  // namespace plast
