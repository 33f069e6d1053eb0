// rows.hpp — what the row operators over fp32, fp16 and bf16 share: where a row of strided leading axes starts, a row's
// units of 16 bytes, stores that another XCD's workgroup reads within the launch, and operands that may not share memory.
#pragma once

#include "half_types.hpp"
#include "places.hpp"

namespace plast {

// Where row `r` of the leading axes starts, in elements, in each of K operands.
template <int K>
struct RowMap {
  int rank;
  MagicDiv ext[kMaxRank];
  int64_t st[K][kMaxRank];
};
template <int K>
struct RowAt {
  int64_t at[K];
};
template <int K>
__device__ __forceinline__ RowAt<K> row_at(const RowMap<K> &M, uint32_t r) {
  RowAt<K> a{};
  for (int d = M.rank - 1; d > 0; --d) {
    const uint32_t q = M.ext[d].div(r), i = r - q * M.ext[d].d;
#pragma unroll
    for (int k = 0; k < K; ++k) a.at[k] += int64_t(i) * M.st[k][d];
    r = q;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) a.at[k] += int64_t(r) * M.st[k][0];
  return a;
}

// 16 bytes of a row.
template <class T>
struct Unit {
  static constexpr uint32_t E = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(E)));
  typedef vec any __attribute__((aligned(sizeof(T))));  // at any element's address
  typedef float floats __attribute__((ext_vector_type(E)));
};
template <class T>
__device__ __forceinline__ typename Unit<T>::vec load_unit(const T *p) {
  return __builtin_nontemporal_load(reinterpret_cast<const typename Unit<T>::any *>(p));
}
template <class T>
__device__ __forceinline__ typename Unit<T>::floats to_floats(typename Unit<T>::vec v) {
  return __builtin_convertvector(v, typename Unit<T>::floats);
}
// Holds a unit as it was read: without it the compiler keeps a 16-bit unit's floats, twice the registers, from
// one use to the next.
template <class V>
__device__ __forceinline__ void keep_raw(V &v) {
  typedef uint32_t words __attribute__((ext_vector_type(4)));
  words w = __builtin_bit_cast(words, v);
  asm volatile("" : "+v"(w));
  v = __builtin_bit_cast(V, w);
}

// The XCDs' L2 caches are not coherent: what a workgroup leaves for another goes past them, store by store (a
// fence would write back and drop the whole cache: 46 us instead of 9 with 384 workgroups).
template <class V>
__device__ __forceinline__ void put_shared(V *p, V v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class V>
__device__ __forceinline__ V get_shared(const V *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

inline bool f32_vector(const Tensor *t, uint64_t n) {
  return t && t->device == GPU && t->dtype == FLOAT32 && numel(t) == n && contiguous(t) && (t->data || n == 0);
}

// An operand that is written, and whether it lies apart from others: reported where one shares memory with it.
struct Operand {
  const char *name;
  const Tensor *t;
  Span span;
  Operand(const char *name, const Tensor *t) : name(name), t(t), span(t) {}
};
inline bool apart(const Operand &written, std::initializer_list<const Operand *> others, const char *where) {
  for (const Operand *o : others)
    if (written.span.meets(o->span) && share_memory(Place(written.t), Place(o->t))) {
      report_error(where, "%s shares memory with %s", written.name, o->name);
      return false;
    }
  return true;
}

}  // namespace plast
