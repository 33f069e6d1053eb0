// Compares share_memory (plast_amd/csrc/places.hpp) with a count of bytes over small strided operands, and takes large
// layouts within its steps: prints "ok" or the first pair that differs, and exits non-zero on failure.
#include <cstdio>
#include <random>
#include <vector>

#include "places.hpp"

using plast::Place;

static Tensor tensor(uint64_t at, std::vector<uint64_t> shape, std::vector<int64_t> strides, DTYPE dtype) {
  Tensor t{};
  t.data = reinterpret_cast<void *>(at);
  t.ndim = shape.size();
  for (size_t d = 0; d < shape.size(); ++d) t.shape[d] = shape[d], t.strides[d] = uint64_t(strides[d]);
  t.dtype = dtype;
  t.device = GPU;
  return t;
}

static void bytes_of(const Tensor &t, std::vector<char> &used) {
  const int bytes = t.dtype == INT64 ? 8 : t.dtype == FLOAT16 || t.dtype == BFLOAT16 ? 2 : 4;
  uint64_t n = 1;
  for (uint64_t d = 0; d < t.ndim; ++d) n *= t.shape[d];
  for (uint64_t i = 0; i < n; ++i) {
    int64_t at = int64_t(reinterpret_cast<uintptr_t>(t.data));
    uint64_t r = i;
    for (uint64_t d = t.ndim; d-- > 0;) at += int64_t(r % t.shape[d]) * int64_t(t.strides[d]) * bytes, r /= t.shape[d];
    for (int e = 0; e < bytes; ++e) used[size_t(at + e)] = 1;
  }
}

static int fail(const char *what, const Tensor &a, const Tensor &b) {
  std::printf("%s:", what);
  for (const Tensor *t : {&a, &b}) {
    std::printf(" at %llu type %d", (unsigned long long)reinterpret_cast<uintptr_t>(t->data), int(t->dtype));
    for (uint64_t d = 0; d < t->ndim; ++d) std::printf(" %llu:%lld", (unsigned long long)t->shape[d], (long long)t->strides[d]);
  }
  std::printf("\n");
  return 1;
}

int main() {
  std::mt19937 rng(1);
  const auto below = [&](int n) { return int(rng() % unsigned(n)); };
  const DTYPE types[] = {FLOAT32, FLOAT16, BFLOAT16, INT32, INT64};
  int shared = 0, apart = 0;
  for (int rep = 0; rep < 20000; ++rep) {
    Tensor t[2];
    const int rank = below(4);
    std::vector<int64_t> first;
    for (int k = 0; k < 2; ++k) {
      std::vector<uint64_t> shape;
      std::vector<int64_t> strides;
      const int r = below(2) ? rank : below(4);
      for (int d = 0; d < r; ++d) {
        shape.push_back(uint64_t(below(6)) + (below(8) ? 1 : 0));
        const int64_t range[] = {3, 9, 24, 60};
        int64_t s = below(int(range[below(4)]));
        if (below(4) == 0) s = -s;
        if (k && r == rank && below(2)) s = first[size_t(d)];  // layouts in common
        strides.push_back(s);
      }
      if (k == 0) first = strides;
      first.resize(8, 5);
      t[k] = tensor(uint64_t(16384 + below(600)), shape, strides, types[below(5)]);
    }
    std::vector<char> used[2];
    bool want = false;
    for (int k = 0; k < 2; ++k) used[k].assign(40000, 0), bytes_of(t[k], used[k]);
    for (size_t i = 0; i < 40000; ++i) want = want || (used[0][i] && used[1][i]);
    if (plast::share_memory(Place(&t[0]), Place(&t[1])) != want) return fail(want ? "not seen" : "seen", t[0], t[1]);
    if (plast::share_memory(Place(&t[1]), Place(&t[0])) != want) return fail("not the same the other way", t[0], t[1]);
    if (want && !plast::Span(&t[0]).meets(plast::Span(&t[1]))) return fail("spans do not meet", t[0], t[1]);
    (want ? shared : apart) += 1;
  }
  if (shared < 2000 || apart < 2000) return std::printf("%d shared, %d apart\n", shared, apart), 1;

  // large layouts: told apart, or seen, in a few steps
  struct { const char *what; Tensor a, b; bool want; } large[] = {
      {"halves of a projection", tensor(1 << 20, {64, 65536, 1000}, {131072000, 2000, 1}, BFLOAT16),
       tensor((1 << 20) + 2000, {64, 65536, 1000}, {131072000, 2000, 1}, BFLOAT16), false},
      {"halves that overlap by an element", tensor(1 << 20, {64, 65536, 1001}, {131072000, 2000, 1}, BFLOAT16),
       tensor((1 << 20) + 2000, {64, 65536, 1000}, {131072000, 2000, 1}, BFLOAT16), true},
      {"the last row behind the first", tensor(1 << 20, {1 << 30, 16}, {16, 1}, FLOAT32),
       tensor((uint64_t(1) << 20) + (uint64_t(64) << 30) - 4, {1 << 30, 16}, {16, 1}, FLOAT32), true},
      {"one behind the other", tensor(1 << 20, {1 << 30, 16}, {16, 1}, FLOAT32),
       tensor((uint64_t(1) << 20) + (uint64_t(64) << 30), {1 << 30, 16}, {16, 1}, FLOAT32), false},
      {"a vector between rows", tensor(1 << 20, {1000000, 100}, {1000, 1}, FLOAT32),
       tensor((1 << 20) + 4000 * 777 + 400, {900}, {1}, FLOAT32), false},
      {"a vector into a row", tensor(1 << 20, {1000000, 100}, {1000, 1}, FLOAT32),
       tensor((1 << 20) + 4000 * 777 + 400, {901}, {1}, FLOAT32), true},
      {"parts of a batch's buffer", tensor(1 << 20, {10000, 300, 64}, {300 * 192, 64, 1}, FLOAT32),
       tensor((1 << 20) + 300 * 64 * 4, {10000, 300, 64}, {300 * 192, 128, 1}, FLOAT32), false},
      {"a row repeated", tensor(1 << 20, {1 << 20, 64}, {0, 1}, FLOAT32), tensor((1 << 20) + 256, {1 << 20, 64}, {64, 1}, FLOAT32), false},
      {"steps that cannot be told apart in time", tensor(1 << 20, {1 << 20, 1}, {1000, 1}, FLOAT32),
       tensor((1 << 20) + 4, {1 << 20, 1}, {998, 1}, FLOAT32), true},
  };
  for (auto &c : large)
    if (plast::share_memory(Place(&c.a), Place(&c.b)) != c.want || plast::share_memory(Place(&c.b), Place(&c.a)) != c.want)
      return fail(c.what, c.a, c.b);
  std::printf("ok\n");
  return 0;
}
