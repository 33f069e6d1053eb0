// gated_recurrence.hip — the gated linear recurrence along a sequence, each channel by itself, and its gradients:
//   a = sigmoid(f),  z = 1 - a,  h[t] = a[t] h[t-1] + z[t] v[t],
//   dh[t] = dy[t] + a[t+1] dh[t+1],  dv = z dh,  df = dh (h[t-1] - v) a z,  dh[-1] = a[0] dh[0].
//
// With e = exp(-|f|), the larger of a and z is 1 / (1 + e) and the smaller e / (1 + e), each to some 4e-7 of itself in fp32 (Gate):
// next to 1 the larger has lost what the smaller holds. A step multiplies the state by a, whose rounding would add up over a long memory
// if steps were all there is: so runs of eight steps are short cuts of their own, which take what they do to a state from the
// smaller sides where those count (Share), and every run starts from there.
// A product with a factor of 0 is 0 whatever the other factor is (v_mul_legacy_f32): a gate so far out that one side is 0
// selects, and lets no NaN through.
//
// A sequence is cut into tiles of steps, a workgroup each, so that a few long ones fill the card, and read once: a tile's share and
// what it adds are left for those behind it, and the state that it starts with comes from those before it within the same launch.
// That wait, a tile's loads, its two passes and its stores follow one another, and the tiles that a CU holds hide it in part: forward
// [1, 65536, 1024] in bf16 99 us, 4.2 TB/s, vector units 42% busy; [8, 4096, 2048] 90 us, 4.8 TB/s, 50%; backward 150 us, 4.8 TB/s, 53%.
// States from two launches more (shares alone, then all again) would read f and v twice.
#include <atomic>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "rows.hpp"

namespace plast {
namespace {

constexpr uint32_t kChunk = PLAST_RECURRENCE_CHUNK;

// A sequence operand: strides of the batch and of time, in elements.
template <class P>
struct Seq {
  P p;
  int64_t b, t;
};
struct ScanArgs {
  Seq<const char *> f, v, dy;
  Seq<char *> h, df, dv;
  const float *initial, *dlast;
  const int32_t *lengths;
  float *last, *states, *dinitial;
  uint32_t batch, length, width, chunks;
  bool past;  // what is read is more than the last-level cache takes
};

extern "C" __device__ float mul_legacy(float, float) __asm("llvm.amdgcn.fmul.legacy");

// Both sides of a gate that is held as T. e = 2^x with x = -|f| log2(e) rounded to fp32, which alone would be off by half a step of x:
// 1e-6 of e at |f| = 20, 4e-6 at 80. What x ln 2 misses of -|f|, t, brings it back, as 2^x (1 + t); t is NaN where f is infinite and 2^x
// is 0, and 1 instead. Sequences in 16 bits go without t (the states in fp32 beside them too): it is a hundredth of their own rounding at
// most, and forward and backward of [8, 4096, 2048] in bf16 takes 243 us with it instead of 237, of [5, 3001, 1003] in fp32 112 instead of 111.
template <class T>
struct Gate {
  float a, z;
  __device__ __forceinline__ explicit Gate(float f) {
    const float x = -1.44269504f * fabsf(f);
    float e = __builtin_amdgcn_exp2f(x);
    if constexpr (sizeof(T) == 4) {
      float t = __builtin_fmaf(x, -0.693147182f, -fabsf(f));  // ln 2 in two parts
      t = __builtin_fmaf(x, 1.90465430e-9f, t);
      e = __builtin_fmaf(e, __builtin_fminf(t, 1.0f), e);
    }
    const float large = __builtin_amdgcn_rcpf(1.0f + e), small = e * large;
    const bool keep = f > 0.0f;
    a = keep ? large : small;
    z = keep ? small : large;
  }
};
constexpr float kHold = __builtin_huge_valf();  // the gate that leaves a state as it is: a is 1, z is 0

// What a run of steps does to the state x before it: x keeps a share and something is added. Of the share both are kept, A and
// its complement C: a long memory's A next to 1 has lost the digits of C that count, a short one's C those of A. `code` is the one
// that counts, A with the sign bit set; -0 for a run with a gate that lets nothing through. A product below fp32's range is not
// that: what it multiplies may be NaN.
struct Share {
  float a = 1.0f, c = 0.0f;
  bool shut = false;
  __device__ __forceinline__ void step(float ga, float gz) {
    c = __builtin_fmaf(ga, c, gz);
    a *= ga;
    shut = shut || ga == 0.0f;
  }
  __device__ __forceinline__ float code() const {
    return shut ? -0.0f : c < 0.9375f ? c : -__builtin_elementwise_maximum(a, 0x1p-149f);  // NaN stays
  }
  // the share of this run and one behind it
  __device__ __forceinline__ void join(float code) {
    const bool is_a = __builtin_signbit(code);
    const float m = fabsf(code), r = 1.0f - m;
    c = __builtin_fmaf(is_a ? r : m, 1.0f - c, c);
    a *= is_a ? m : r;
    shut = shut || (is_a && m == 0.0f);
  }
};
__device__ __forceinline__ float apply(float code, float plus, float x) {
  if (!__builtin_signbit(code)) return plus + __builtin_fmaf(-code, x, x);
  return code == 0.0f ? plus : __builtin_fmaf(-code, x, plus);
}

__device__ __forceinline__ f4 apply(f4 code, f4 plus, f4 x) {
  f4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = apply(code[e], plus[e], x[e]);
  return y;
}

__device__ __forceinline__ uint32_t live_steps(const ScanArgs &A, uint32_t b) {
  const int32_t n = A.lengths[b];
  return n < 0 ? 0 : uint32_t(n) < A.length ? uint32_t(n) : A.length;
}

// Four channels of a step; n of them lie inside the row.
template <class T>
struct Quad {
  typedef T vec __attribute__((ext_vector_type(4)));
  typedef vec any __attribute__((aligned(sizeof(T))));
};
template <class T>
__device__ __forceinline__ typename Quad<T>::vec load_quad(const T *p, int n, float otherwise = 0.0f) {
  if (n >= 4) return *reinterpret_cast<const typename Quad<T>::any *>(p);
  typename Quad<T>::vec v = T(otherwise);
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < n) v[e] = p[e];
  return v;
}
template <class T>
__device__ __forceinline__ void store_quad(T *p, f4 f, int n) {
  const typename Quad<T>::vec v = __builtin_convertvector(f, typename Quad<T>::vec);
  if (n >= 4) {
    __builtin_nontemporal_store(v, reinterpret_cast<typename Quad<T>::any *>(p));
    return;
  }
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < n) p[e] = v[e];
}
// A whole quad past the caches, and quads as above, at a lane's offset in bytes from a step's address, which is the same for all
// lanes.
template <class T>
__device__ __forceinline__ typename Quad<T>::vec load_past(const void *step, uint32_t offset) {
  return __builtin_nontemporal_load(reinterpret_cast<const typename Quad<T>::any *>(static_cast<const char *>(step) + offset));
}
template <class T>
__device__ __forceinline__ typename Quad<T>::vec load_at(const void *step, uint32_t offset, int n, float otherwise = 0.0f) {
  return load_quad(reinterpret_cast<const T *>(static_cast<const char *>(step) + offset), n, otherwise);
}
// A lane's quad that was read `back` channels before where it lies, so that it ends with the row: what is in the row, and
// `otherwise`. Reads under a branch each wait for the one before; these are all on their way at once: forward / backward of
// [5, 3001, 1003] in fp32 37.8 / 86 -> 35.6 / 78 us, in bf16 37.7 / 77 -> 32.9 / 63, of [5, 10866, 229] in bf16 42.9 / 84 -> 37.7 / 64.
template <class T>
__device__ __forceinline__ void move_quad(typename Quad<T>::vec &q, int back, float otherwise) {
  const typename Quad<T>::vec was = q;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    T v = back == 0 ? was[e] : T(otherwise);
#pragma unroll
    for (int m = 1; m < 4 - e; ++m) v = back == m ? was[e + m] : v;
    q[e] = v;
  }
}
template <class T>
__device__ __forceinline__ void store_at(void *step, uint32_t offset, f4 f, int n) {
  store_quad(reinterpret_cast<T *>(static_cast<char *>(step) + offset), f, n);
}
template <class T>
__device__ __forceinline__ f4 to_f4(typename Quad<T>::vec v) {
  return __builtin_convertvector(v, f4);
}

// Holds quads as they were read from one pass to the next: without it the compiler keeps their floats, and what was worked out
// of them, beside them.
template <class V, uint32_t N>
__device__ __forceinline__ void keep_raw(V (&v)[N]) {
  typedef uint32_t words __attribute__((ext_vector_type(sizeof(V) / 4)));
#pragma unroll
  for (uint32_t k = 0; k < N; ++k) {
    words w = __builtin_bit_cast(words, v[k]);
    asm volatile("" : "+v"(w));
    v[k] = __builtin_bit_cast(V, w);
  }
}

// ------------------------------------------------------------------------- tiles

// A tile is TILE steps (one kChunk or several) of some channels: lanes across, four channels each, and slices of a few steps, a slice
// a lane's. Every lane finds its slice's share and what it adds from a state of 0, the slices' are joined in LDS, and each lane goes
// through its steps again from the state that its slice starts with.
template <uint32_t ACROSS, uint32_t STEPS, uint32_t TILE, uint32_t WAVES>
struct Shape {
  static constexpr uint32_t kAcross = ACROSS, kSteps = STEPS, kTile = TILE, kWidth = 4 * ACROSS, kSlices = TILE / STEPS;
  static constexpr uint32_t kLanes = ACROSS * kSlices, kWaves = WAVES;  // waves that share a SIMD
  static constexpr uint32_t kChunkSlices = kChunk / STEPS;
  static_assert(kTile % kChunk == 0 && kChunk % kSteps == 0 && kWidth % 64 == 0, "whole chunks, slices and waves");
};

// What a tile leaves of 64 channels for those behind it: `plus` and `code` of the tile alone, and the state after it. A word's
// upper half is the launch's tag where the word is there, so each word counts by itself.
struct Record {
  uint64_t code[64], plus[64], state[64];
};
constexpr uint32_t kMostGets = 1u << 20;
struct Look {
  Record *records;  // [tiles of a sequence][64 channels of the columns of tiles]
  uint32_t tiles, tag, most;
  __device__ __forceinline__ void put(uint64_t *p, float v) const { put_shared(p, uint64_t(tag) << 32 | __float_as_uint(v)); }
  __device__ __forceinline__ bool there(uint64_t w) const { return uint32_t(w >> 32) == tag; }
  // A word that has been sent, and may be under way. It comes, but where a launch on another stream writes the same records: NaN.
  __device__ __forceinline__ float get(const uint64_t *p) const {
    for (uint32_t i = 0; i < kMostGets; ++i) {
      const uint64_t w = get_shared(p);
      if (there(w)) return __uint_as_float(uint32_t(w));
    }
    return __builtin_nanf("");
  }
};

__global__ __launch_bounds__(256) void clear_kernel(uint64_t *p, uint64_t n) {
  const uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) p[i] = 0;
}

__global__ __launch_bounds__(256) void copy_kernel(float *to, const float *from, uint64_t n) {
  const uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) to[i] = from[i];
}

// Which tile a workgroup works on. Workgroups are dispatched in their order, round robin over the eight XCDs: an XCD's take
// columns of its own (`each`; 0: all take all), tile by tile, so that what lies side by side is read side by side.
struct Tile {
  uint32_t i, column, b, c0, t0, end;  // i: its number in the sequence; c0, t0: first channel and step; end: steps that are there
  bool none, dead, whole, steps;  // no tile; padding alone; all of its steps and channels there, so that it needs no bounds; all of
                                  // its steps, and a quad of channels or more
};
template <class S, bool BACK>
__device__ __forceinline__ Tile tile_at(const ScanArgs &A, const Look &L, uint32_t across, uint32_t each) {
  const uint32_t columns = A.batch * across, i = blockIdx.x;
  Tile t;
  if (each) {
    t.i = i / 8 / each;
    t.column = i % 8 * each + i / 8 % each;
  } else {
    t.i = i / columns;
    t.column = i - t.i * columns;
  }
  t.none = t.column >= columns;
  if (t.none) return t;
  if (BACK) t.i = L.tiles - 1 - t.i;
  t.b = t.column / across;
  t.c0 = (t.column - t.b * across) * S::kWidth;
  t.t0 = t.i * S::kTile;
  t.end = live_steps(A, t.b);
  t.dead = t.i > 0 && t.t0 >= t.end;
  t.steps = t.t0 + S::kTile <= t.end && t.c0 + 4 <= A.width;
  t.whole = t.steps && t.c0 + S::kWidth <= A.width;
  return t;
}
// Where a tile lies in a sequence operand: the address of its step k, and the offset from there of a lane whose slice starts
// `first` steps into the tile and whose channels are `c` into it.
template <class T, class P>
struct TileSeq {
  P p;
  int64_t step;
  uint32_t offset;
  __device__ __forceinline__ TileSeq(const Seq<P> &s, const Tile &t, uint32_t first, uint32_t c) {
    p = s.p + (int64_t(t.b) * s.b + int64_t(t.t0) * s.t + t.c0) * int64_t(sizeof(T));
    step = s.t * int64_t(sizeof(T));
    offset = (first * uint32_t(s.t) + c) * uint32_t(sizeof(T));
  }
  __device__ __forceinline__ P at(uint32_t k) const { return p + step * k; }
};

// A channel's tile `i` worked out by one lane, bit for bit as its own workgroup does.
template <class T, class S, bool BACK>
__device__ __forceinline__ void tile_share(const ScanArgs &A, const Tile &t, uint32_t tile, uint32_t channel, float &code, float &plus) {
  constexpr uint32_t kSlices = S::kSlices, kSteps = S::kSteps;
  Share joined;
  float all = 0.0f;
  const uint64_t at = uint64_t(t.b) * A.width + channel;
#pragma unroll 1
  for (uint32_t i = 0; i < kSlices; ++i) {
    const uint32_t t0 = tile * S::kTile + (BACK ? kSlices - 1 - i : i) * kSteps;
    float keep[kSteps], sum = 0.0f;
    Share share;
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      const bool live = t0 + k < t.end && channel < A.width;
      const T *f = reinterpret_cast<const T *>(A.f.p) + int64_t(t.b) * A.f.b + int64_t(t0 + k) * A.f.t + channel;
      const T *v = reinterpret_cast<const T *>(A.v.p) + int64_t(t.b) * A.v.b + int64_t(t0 + k) * A.v.t + channel;
      const Gate<T> g(live ? float(*f) : kHold);
      keep[k] = g.a;
      share.step(g.a, g.z);
      if (!BACK) sum = mul_legacy(g.a, sum) + mul_legacy(g.z, live ? float(*v) : 0.0f);
    }
    if (BACK)
#pragma unroll
      for (uint32_t k = kSteps; k-- > 0;) {
        const bool live = t0 + k < t.end && channel < A.width;
        const T *dy = reinterpret_cast<const T *>(A.dy.p) + int64_t(t.b) * A.dy.b + int64_t(t0 + k) * A.dy.t + channel;
        float d = live && A.dy.p ? float(*dy) : 0.0f;
        if (t0 + k + 1 == t.end && A.dlast && channel < A.width) d += A.dlast[at];
        sum = mul_legacy(keep[k], sum + d);
      }
    const float c = share.code();
    joined.join(c);
    all = apply(c, sum, all);
  }
  code = joined.code();
  plus = all;
}

// The state that a tile starts with, a lane a channel of a wave's 64: of the `n` tiles before it (`step` records apart) the
// nearest whose state is there is found, and the shares of those between are applied to it one after the other, as they
// themselves do: the bits do not depend on which it was. One load looks at 32 tiles, a word of each: looking at all of what a
// few of them leave, again and again, took half of the memory's rate.
// Workgroups start in the order of their tiles, so those before are at work, and each leaves its own share before it waits for
// anything. Should one not come, as nothing promises that order, its share is worked out here after L.most looks: every wait ends.
template <class T, class S, bool BACK>
__device__ __forceinline__ float look_back(const ScanArgs &A, const Look &L, const Tile &t, uint32_t channel, Record *mine,
                                           int64_t step, uint32_t n, uint32_t lane, uint64_t ready, float code, float plus) {
  if (__all(L.there(ready))) return __uint_as_float(uint32_t(ready));
  L.put(&mine->code[lane], code);
  L.put(&mine->plus[lane], plus);
  uint32_t d0 = 1, looks = 0;  // the nearest tile of a look is d0 before this one
  for (;;) {
    const uint32_t at = d0 + (lane & 31);
    const Record *r = mine - step * int64_t(at < n ? at : n);
    const uint64_t seen = __ballot(L.there(get_shared(lane < 32 ? &r->code[0] : &r->state[0])));
    const uint32_t shares = uint32_t(seen), states = uint32_t(seen >> 32);
    const uint32_t known = __builtin_ctzll(~uint64_t(shares));  // tiles whose shares are there, up to the first that is not
    if (states && uint32_t(__builtin_ctz(states)) <= known) {
      d0 += __builtin_ctz(states);
      break;
    }
    if (known == 32 && d0 + 32 <= n) {
      d0 += 32;
    } else if (++looks < L.most) {
      __builtin_amdgcn_s_sleep(1);
    } else {  // the first tile has a state alone
      const uint32_t d = d0 + known < n ? d0 + known : n;
      Record *late = mine - step * int64_t(d);
      float own_code, own_plus;
      tile_share<T, S, BACK>(A, t, BACK ? t.i + d : t.i - d, channel, own_code, own_plus);
      if (BACK ? (t.i + d + 1) * S::kTile >= t.end : t.i == d) {
        const float from = !BACK && channel < A.width ? A.initial[uint64_t(t.b) * A.width + channel] : 0.0f;
        L.put(&late->state[lane], apply(own_code, own_plus, from));
      } else {
        L.put(&late->code[lane], own_code);
        L.put(&late->plus[lane], own_plus);
      }
    }
  }
  float x = L.get(&(mine - step * int64_t(d0))->state[lane]);
  constexpr uint32_t W = 4;
  uint32_t turns = 0;
  for (uint32_t d = d0 - 1; d > 0;) {
    if (++turns == kMostGets) return __builtin_nanf("");  // as above
    uint64_t c[W], p[W];
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
      const Record *r = mine - step * int64_t(d > w ? d - w : 1);
      c[w] = get_shared(&r->code[lane]);
      p[w] = get_shared(&r->plus[lane]);
    }
    uint32_t done = 0;
    bool there = true;
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
      there = there && w < d && __all(L.there(c[w]) && L.there(p[w]));
      if (there) x = apply(__uint_as_float(uint32_t(c[w])), __uint_as_float(uint32_t(p[w])), x), ++done;
    }
    d -= done;
  }
  return x;
}

template <class T, class S, bool MANY>
__global__ __launch_bounds__(S::kLanes, S::kWaves) void fwd_kernel(ScanArgs A, Look L, uint32_t tiles_across, uint32_t each) {
  constexpr uint32_t kAcross = S::kAcross, kSteps = S::kSteps, kSlices = S::kSlices, kTileWidth = S::kWidth;
  __shared__ __align__(16) float codes[kSlices][kTileWidth], plus[kSlices][kTileWidth], starts[kTileWidth];
  const Tile t = tile_at<S, false>(A, L, tiles_across, each);
  if (t.none) return;
  const uint32_t across = 4 * (threadIdx.x & (kAcross - 1)), slice = threadIdx.x / kAcross;
  const uint32_t c = t.c0 + across, t0 = t.t0 + slice * kSteps;
  const int n = int(A.width) - int(c);
  const TileSeq<T, char *> y(A.h, t, slice * kSteps, across);
  if (t.dead) {
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k)
      if (t0 + k < A.length) store_at<T>(y.at(k), y.offset, f4(0.0f), n);
    return;
  }
  const TileSeq<T, const char *> f(A.f, t, slice * kSteps, across), v(A.v, t, slice * kSteps, across);
  typename Quad<T>::vec gates[kSteps], val[kSteps];
  // The path of long operands stays in line: without the hint the forward pass of [1, 65536, 1024] in bf16 takes 106 us instead of 102.
  if (__builtin_expect(t.whole && A.past, 1)) {
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      gates[k] = load_past<T>(f.at(k), f.offset);
      val[k] = load_past<T>(v.at(k), v.offset);
    }
  } else if (t.whole) {
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      gates[k] = load_at<T>(f.at(k), f.offset, 4);
      val[k] = load_at<T>(v.at(k), v.offset, 4);
    }
  } else if (t.steps) {  // quads that reach beyond the row are read from inside it, without branches
    const int back = n >= 4 ? 0 : 4 - n;
    const uint32_t off = uint32_t(back) * uint32_t(sizeof(T));
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      gates[k] = load_at<T>(f.at(k), f.offset - off, 4);
      val[k] = load_at<T>(v.at(k), v.offset - off, 4);
    }
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      move_quad<T>(gates[k], back, kHold);
      move_quad<T>(val[k], back, 0.0f);
    }
  } else {
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      const int m = t0 + k < t.end ? n : 0;
      gates[k] = load_at<T>(f.at(k), f.offset, m, kHold);
      val[k] = load_at<T>(v.at(k), v.offset, m);
    }
  }
  // the first waves' lanes are the tile's channels while the slices are joined
  const uint32_t lane = threadIdx.x, channel = t.c0 + lane;
  const bool joins = lane < kTileWidth, inside = channel < A.width;
  const int64_t columns = int64_t(A.batch) * tiles_across * (kTileWidth / 64);
  Record *mine = MANY ? L.records + t.i * columns + t.column * (kTileWidth / 64) + lane / 64 : nullptr;
  uint64_t ready = 0;
  float start = 0.0f;
  if (joins) {
    if (MANY && t.i > 0) ready = get_shared(&(mine - columns)->state[lane & 63]);
    else if (inside) start = A.initial[uint64_t(t.b) * A.width + channel];
  }
  f4 keep[kSteps], add[kSteps], sum = 0.0f;
  Share share[4];
#pragma unroll
  for (uint32_t k = 0; k < kSteps; ++k) {
    const f4 x = to_f4<T>(gates[k]), u = to_f4<T>(val[k]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const Gate<T> g(x[e]);
      keep[k][e] = g.a;
      add[k][e] = mul_legacy(g.z, u[e]);
      share[e].step(g.a, g.z);
      sum[e] = mul_legacy(g.a, sum[e]) + add[k][e];
    }
  }
  f4 code;
#pragma unroll
  for (int e = 0; e < 4; ++e) code[e] = share[e].code();
  *reinterpret_cast<f4 *>(&codes[slice][across]) = code;
  *reinterpret_cast<f4 *>(&plus[slice][across]) = sum;
  __syncthreads();
  if (joins) {  // before each slice: the share of those before it and what they add
    Share joined;
    float all = 0.0f;
#pragma unroll 8
    for (uint32_t i = 0; i < kSlices; ++i) {
      const float one = codes[i][lane], more = plus[i][lane];
      codes[i][lane] = joined.code();
      plus[i][lane] = all;
      joined.join(one);
      all = apply(one, more, all);
    }
    if constexpr (MANY) {
      if (t.i > 0) start = look_back<T, S, false>(A, L, t, channel, mine, columns, t.i, lane & 63, ready, joined.code(), all);
      L.put(&mine->state[lane & 63], apply(joined.code(), all, start));
    }
    if (t.end == 0 && inside) A.last[uint64_t(t.b) * A.width + channel] = start;
    starts[lane] = start;
  }
  __syncthreads();
  f4 h = apply(*reinterpret_cast<const f4 *>(&codes[slice][across]), *reinterpret_cast<const f4 *>(&plus[slice][across]),
               *reinterpret_cast<const f4 *>(&starts[across]));
  if (A.states && slice % S::kChunkSlices == 0 && t0 < A.length)
    store_quad<float>(A.states + (uint64_t(t.b) * A.chunks + t0 / kChunk) * A.width + c, h, n);
  if (t.whole) {
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = mul_legacy(keep[k][e], h[e]) + add[k][e];
      store_at<T>(y.at(k), y.offset, h, 4);
    }
    if (t0 + kSteps == t.end) store_quad<float>(A.last + uint64_t(t.b) * A.width + c, h, 4);
    return;
  }
#pragma unroll
  for (uint32_t k = 0; k < kSteps; ++k) {
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = mul_legacy(keep[k][e], h[e]) + add[k][e];
    if (t0 + k < A.length) store_at<T>(y.at(k), y.offset, t0 + k < t.end ? h : f4(0.0f), n);
    if (t0 + k + 1 == t.end) store_quad<float>(A.last + uint64_t(t.b) * A.width + c, h, n);
  }
}

template <class T, bool ADD>
__device__ __forceinline__ void put_at(char *step, uint32_t offset, f4 f, int n) {
  if constexpr (ADD) f += to_f4<T>(load_at<T>(step, offset, n));
  store_at<T>(step, offset, f, n);
}

template <class T, class S, bool ADD, bool MANY>
__global__ __launch_bounds__(S::kLanes, S::kWaves) void bwd_kernel(ScanArgs A, Look L, uint32_t tiles_across, uint32_t each) {
  constexpr uint32_t kAcross = S::kAcross, kSteps = S::kSteps, kSlices = S::kSlices, kTileWidth = S::kWidth;
  __shared__ __align__(16) float codes[kSlices][kTileWidth], plus[kSlices][kTileWidth], back[kSlices][kTileWidth];
  __shared__ __align__(16) float after[kSlices][kTileWidth], starts[kTileWidth];
  const Tile t = tile_at<S, true>(A, L, tiles_across, each);
  if (t.none) return;
  const uint32_t across = 4 * (threadIdx.x & (kAcross - 1)), slice = threadIdx.x / kAcross;
  const uint32_t c = t.c0 + across, t0 = t.t0 + slice * kSteps;
  const int n = int(A.width) - int(c);
  const TileSeq<T, char *> df(A.df, t, slice * kSteps, across), dv(A.dv, t, slice * kSteps, across);
  if (t.dead) {
    if (!ADD)
#pragma unroll
      for (uint32_t k = 0; k < kSteps; ++k)
        if (t0 + k < A.length) {
          if (A.df.p) store_at<T>(df.at(k), df.offset, f4(0.0f), n);
          if (A.dv.p) store_at<T>(dv.at(k), dv.offset, f4(0.0f), n);
        }
    return;
  }
  const TileSeq<T, const char *> f(A.f, t, slice * kSteps, across), v(A.v, t, slice * kSteps, across),
      dy(A.dy, t, slice * kSteps, across);
  typename Quad<T>::vec gates[kSteps], val[kSteps], up[kSteps];
  const bool whole = t.whole && A.dy.p && A.df.p && A.dv.p;
  if (__builtin_expect(whole && A.past, 1)) {
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      gates[k] = load_past<T>(f.at(k), f.offset);
      val[k] = load_past<T>(v.at(k), v.offset);
      up[k] = load_past<T>(dy.at(k), dy.offset);
    }
  } else if (whole) {
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      gates[k] = load_at<T>(f.at(k), f.offset, 4);
      val[k] = load_at<T>(v.at(k), v.offset, 4);
      up[k] = load_at<T>(dy.at(k), dy.offset, 4);
    }
  } else if (t.steps && A.dy.p) {  // as forward
    const int back = n >= 4 ? 0 : 4 - n;
    const uint32_t off = uint32_t(back) * uint32_t(sizeof(T));
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      gates[k] = load_at<T>(f.at(k), f.offset - off, 4);
      val[k] = load_at<T>(v.at(k), v.offset - off, 4);
      up[k] = load_at<T>(dy.at(k), dy.offset - off, 4);
    }
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      move_quad<T>(gates[k], back, kHold);
      move_quad<T>(val[k], back, 0.0f);
      move_quad<T>(up[k], back, 0.0f);
    }
  } else {
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      const int m = t0 + k < t.end ? n : 0;
      gates[k] = load_at<T>(f.at(k), f.offset, m, kHold);
      val[k] = load_at<T>(v.at(k), v.offset, m);
      up[k] = load_at<T>(dy.at(k), dy.offset, A.dy.p ? m : 0);
    }
  }
  // the first waves join the slices forward, the next ones from the end
  const uint32_t lane = threadIdx.x & (kTileWidth - 1), channel = t.c0 + lane, role = threadIdx.x / kTileWidth;
  const bool inside = channel < A.width, last = t.t0 + S::kTile >= t.end;  // last: nothing comes from behind
  const int64_t columns = int64_t(A.batch) * tiles_across * (kTileWidth / 64);
  Record *mine = MANY ? L.records + (L.tiles - 1 - t.i) * columns + t.column * (kTileWidth / 64) + lane / 64 : nullptr;
  const uint64_t state_at = uint64_t(t.b) * A.width + channel;
  float start = 0.0f;
  uint64_t ready = 0;
  if (role == 0 && inside && t.end) start = A.states[(uint64_t(t.b) * A.chunks + t.t0 / kChunk) * A.width + channel];
  if (MANY && role == 1 && !last) ready = get_shared(&(mine - columns)->state[lane & 63]);
  f4 dlast = 0.0f;
  if (A.dlast && t.end && t0 < t.end && t.end <= t0 + kSteps) dlast = load_quad<float>(A.dlast + uint64_t(t.b) * A.width + c, n);
  f4 keep[kSteps], into[kSteps], sum = 0.0f, rev = 0.0f;
  Share share[4];
#pragma unroll
  for (uint32_t k = 0; k < kSteps; ++k) {
    const f4 x = to_f4<T>(gates[k]), u = to_f4<T>(val[k]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const Gate<T> g(x[e]);
      keep[k][e] = g.a;
      into[k][e] = g.z;
      share[e].step(g.a, g.z);
      sum[e] = mul_legacy(g.a, sum[e]) + mul_legacy(g.z, u[e]);
    }
  }
#pragma unroll
  for (uint32_t k = kSteps; k-- > 0;) {
    f4 d = to_f4<T>(up[k]);
    if (t0 + k + 1 == t.end) d += dlast;
#pragma unroll
    for (int e = 0; e < 4; ++e) rev[e] = mul_legacy(keep[k][e], rev[e] + d[e]);
  }
  f4 code;
#pragma unroll
  for (int e = 0; e < 4; ++e) code[e] = share[e].code();
  *reinterpret_cast<f4 *>(&codes[slice][across]) = code;
  *reinterpret_cast<f4 *>(&plus[slice][across]) = sum;
  *reinterpret_cast<f4 *>(&back[slice][across]) = rev;
  __syncthreads();
  keep_raw(val);
  keep_raw(up);
  if (role == 0) {
#pragma unroll 8
    for (uint32_t i = 0; i < kSlices; ++i) {
      const float after = apply(codes[i][lane], plus[i][lane], start);
      plus[i][lane] = start;
      start = after;
    }
  } else if (role == 1) {  // behind each slice: the share of those behind it and what they add
    float from = 0.0f;  // a dh of the step behind the tile
    Share joined;
    float all = 0.0f;
#pragma unroll 8
    for (uint32_t i = kSlices; i-- > 0;) {
      const float one = codes[i][lane], more = back[i][lane];
      after[i][lane] = joined.code();
      back[i][lane] = all;
      joined.join(one);
      all = apply(one, more, all);
    }
    if constexpr (MANY) {
      if (!last)
        from = look_back<T, S, true>(A, L, t, channel, mine, columns, L.tiles - 1 - t.i, lane & 63, ready, joined.code(), all);
      L.put(&mine->state[lane & 63], apply(joined.code(), all, from));
    }
    starts[lane] = from;
    if (t.i == 0 && A.dinitial && inside) {
      from = t.end ? apply(joined.code(), all, from) : A.dlast ? A.dlast[state_at] : 0.0f;
      A.dinitial[state_at] = ADD ? A.dinitial[state_at] + from : from;
    }
  }
  __syncthreads();
  f4 h = *reinterpret_cast<const f4 *>(&plus[slice][across]);
  f4 d = apply(*reinterpret_cast<const f4 *>(&after[slice][across]), *reinterpret_cast<const f4 *>(&back[slice][across]),
               *reinterpret_cast<const f4 *>(&starts[across]));
  f4 dh[kSteps];
  keep_raw(up);
  keep_raw(val);
#pragma unroll
  for (uint32_t k = kSteps; k-- > 0;) {
    f4 u = to_f4<T>(up[k]);
    if (t0 + k + 1 == t.end) u += dlast;
    dh[k] = d + u;
#pragma unroll
    for (int e = 0; e < 4; ++e) d[e] = mul_legacy(keep[k][e], dh[k][e]);
  }
  const auto gradients = [&](uint32_t k, f4 &to_f, f4 &to_v) {
    const f4 u = to_f4<T>(val[k]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      to_v[e] = mul_legacy(into[k][e], dh[k][e]);
      to_f[e] = mul_legacy(keep[k][e] * into[k][e], dh[k][e] * (h[e] - u[e]));
      h[e] = mul_legacy(keep[k][e], h[e]) + mul_legacy(into[k][e], u[e]);
    }
  };
  if (whole) {
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      f4 to_f, to_v;
      gradients(k, to_f, to_v);
      put_at<T, ADD>(df.at(k), df.offset, to_f, 4);
      put_at<T, ADD>(dv.at(k), dv.offset, to_v, 4);
    }
    return;
  }
#pragma unroll
  for (uint32_t k = 0; k < kSteps; ++k) {
    f4 to_f, to_v;
    gradients(k, to_f, to_v);
    if (t0 + k >= t.end) to_f = to_v = f4(0.0f);
    if (t0 + k < (ADD ? t.end : A.length)) {
      if (A.df.p) put_at<T, ADD>(df.at(k), df.offset, to_f, n);
      if (A.dv.p) put_at<T, ADD>(dv.at(k), dv.offset, to_v, n);
    }
  }
}

// ------------------------------------------------------------------------- few steps

// A lane four channels, step by step: tokens of a decode batch.
constexpr uint32_t kFewSteps = 16, kFewLanes = 256;
template <class T>
__global__ __launch_bounds__(kFewLanes) void few_kernel(ScanArgs A, uint32_t quads) {
  const uint64_t i = uint64_t(blockIdx.x) * kFewLanes + threadIdx.x;
  if (i >= uint64_t(A.batch) * quads) return;
  const uint32_t b = uint32_t(i / quads), c = 4 * (uint32_t(i) - b * quads), end = live_steps(A, b);
  const int n = int(A.width) - int(c);
  const uint64_t at = uint64_t(b) * A.width + c;
  f4 h = load_quad<float>(A.initial + at, n);
  if (A.states && A.length) store_quad<float>(A.states + at, h, n);
  for (uint32_t t = 0; t < A.length; ++t) {
    if (t < end) {
      const f4 x = to_f4<T>(load_quad<T>(reinterpret_cast<const T *>(A.f.p) + int64_t(b) * A.f.b + int64_t(t) * A.f.t + c, n));
      const f4 u = to_f4<T>(load_quad<T>(reinterpret_cast<const T *>(A.v.p) + int64_t(b) * A.v.b + int64_t(t) * A.v.t + c, n));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Gate<T> g(x[e]);
        h[e] = mul_legacy(g.a, h[e]) + mul_legacy(g.z, u[e]);
      }
    }
    store_quad<T>(reinterpret_cast<T *>(A.h.p) + int64_t(b) * A.h.b + int64_t(t) * A.h.t + c, t < end ? h : f4(0.0f), n);
  }
  store_quad<float>(A.last + at, h, n);
}

// ------------------------------------------------------------------------- host

// A lane's offset in a tile has 32 bits.
constexpr uint64_t kMostStep = uint64_t(1) << 22;
bool sequence(const Tensor *t, const Tensor *f) {
  return t && t->device == GPU && t->dtype == f->dtype && same_shape(t, f) && (numel(f) == 0 || t->data) &&
         (f->shape[2] <= 1 || t->strides[2] == 1) && (f->shape[1] <= 1 || t->strides[1] <= kMostStep);
}
template <class P>
Seq<P> seq(const Tensor *t) {
  return {static_cast<P>(t->data), t->shape[0] > 1 ? int64_t(t->strides[0]) : 0, t->shape[1] > 1 ? int64_t(t->strides[1]) : 0};
}

// Checks what both directions take: f, v, lengths, the states that are kept.
bool scan_args(ScanArgs &A, const Tensor *const *in, bool states, const char *where) {
  memset(&A, 0, sizeof A);
  const Tensor *f = in[0], *v = in[1], *initial = in[2], *lengths = in[3], *last = in[4];
  if (!f || !v || !initial || !lengths || !last) {
    report_error(where, "an input is NULL");
    return false;
  }
  if (f->device != GPU || !is_float(f) || f->ndim != 3) {
    report_error(where, "f must be a GPU tensor [batch, time, channels] of FLOAT32, FLOAT16 or BFLOAT16");
    return false;
  }
  const uint64_t B = f->shape[0], L = f->shape[1], D = f->shape[2];
  if (B >= uint64_t(1) << 31 || L >= uint64_t(1) << 31 || D >= uint64_t(1) << 31 || (B && D >= (uint64_t(1) << 32) / B)) {
    report_error(where, "[%llu, %llu, %llu] is not supported", (unsigned long long)B, (unsigned long long)L,
                 (unsigned long long)D);
    return false;
  }
  if (!sequence(f, f) || !sequence(v, f)) {
    report_error(where, "f and v must have one type and shape and a contiguous last axis");
    return false;
  }
  if (!f32_vector(initial, B * D) || !f32_vector(last, B * D)) {
    report_error(where, "the initial and the last state must be contiguous FLOAT32 GPU tensors of %llu elements",
                 (unsigned long long)(B * D));
    return false;
  }
  if (lengths->device != GPU || lengths->dtype != INT32 || numel(lengths) != B || !contiguous(lengths) ||
      (B && !lengths->data)) {
    report_error(where, "lengths must be a contiguous INT32 GPU tensor of %llu elements", (unsigned long long)B);
    return false;
  }
  A.chunks = uint32_t((L + kChunk - 1) / kChunk);
  if (states) {
    if (!f32_vector(in[5], B * A.chunks * D)) {
      report_error(where, "states must be a contiguous FLOAT32 GPU tensor of %llu elements",
                   (unsigned long long)(B * A.chunks * D));
      return false;
    }
    A.states = static_cast<float *>(in[5]->data);
  }
  A.f = seq<const char *>(f);
  A.v = seq<const char *>(v);
  A.initial = static_cast<const float *>(initial->data);
  A.lengths = static_cast<const int32_t *>(lengths->data);
  A.last = static_cast<float *>(last->data);
  A.batch = uint32_t(B);
  A.length = uint32_t(L);
  A.width = uint32_t(D);
  return true;
}

// How often a workgroup looks for a chunk before it works the chunk out itself: some milliseconds.
uint32_t g_most_looks = 4096;
std::atomic<uint32_t> g_tag{1};  // of the last launch over the workspace's records; the graphs' is 1

// The records of a launch over several chunks. Eager launches tag theirs with a number of their own, so that no record of
// another one counts; the slot's records are zeros at first. A graph's replays all have one tag, and clear theirs. `kept` gets room
// for `more` floats beside them.
bool look_at(Look &L, uint64_t records, uint64_t more, float *&kept, const char *where) {
  L.most = g_most_looks;
  const uint64_t bytes = records * sizeof(Record), beside = more * sizeof(float);
  const auto clear = [](void *p, uint64_t n) {
    clear_kernel<<<ceil_div(n / 8, 256), 256, 0, stream()>>>(static_cast<uint64_t *>(p), n / 8);
  };
  if (capturing() && bytes > workspace_bytes(kRecordSlot)) {
    L.records = static_cast<Record *>(partials(bytes + beside, where));
    if (more && L.records) kept = reinterpret_cast<float *>(L.records + records);
  } else if (more) {
    kept = static_cast<float *>(partials(beside, where));
    if (!kept) return false;
  }
  if (capturing()) {
    L.tag = 1;
    if (!L.records) L.records = static_cast<Record *>(workspace(bytes, kRecordSlot));
    if (L.records) clear(L.records, bytes);
  } else {
    L.records = static_cast<Record *>(workspace(bytes, kRecordSlot));
    L.tag = ++g_tag;
    if (L.tag < 2) {  // all numbers have been used
      if (L.records) clear(L.records, workspace_bytes(kRecordSlot));
      g_tag = L.tag = 2;
    }
  }
  return L.records != nullptr;
}
// launch(args, workgroups, records, tiles across a sequence, columns of an XCD)
template <class S, class F>
bool by_tiles(ScanArgs A, const char *where, F &&launch) {
  const uint32_t across = ceil_div(A.width, S::kWidth);
  const uint64_t columns = uint64_t(A.batch) * across;
  // columns that an XCD has more of than another cost time
  const uint64_t each = columns % 8 == 0 || columns >= 128 ? (columns + 7) / 8 : 0;
  Look L{nullptr, A.length > S::kTile ? ceil_div(A.length, S::kTile) : 1, 0, 0};
  const uint64_t blocks = (each ? 8 * each : columns) * L.tiles;
  if (blocks > max_blocks(S::kLanes)) {
    report_error(where, "%llu tiles of %u steps and %u channels are not supported", (unsigned long long)blocks, S::kTile, S::kWidth);
    return false;
  }
  if (L.tiles > 1) {
    // a tile that is worked out by another one's workgroup reads the initial state, whenever that is
    const uint64_t states = A.h.p && A.initial == A.last ? uint64_t(A.batch) * A.width : 0;
    float *kept = nullptr;
    if (!look_at(L, columns * (S::kWidth / 64) * L.tiles, states, kept, where)) return false;
    if (states) {
      copy_kernel<<<ceil_div(states, 256), 256, 0, stream()>>>(kept, A.initial, states);
      A.initial = kept;
    }
  }
  launch(A, unsigned(blocks), L, across, uint32_t(each));
  return true;
}

template <class T, class S>
bool launch_fwd(const ScanArgs &A, const char *where) {
  return by_tiles<S>(A, where, [](const ScanArgs &A, unsigned blocks, const Look &L, uint32_t across, uint32_t each) {
    if constexpr (S::kTile < 256)  // the longest have several
      if (L.tiles == 1) {
        fwd_kernel<T, S, false><<<blocks, S::kLanes, 0, stream()>>>(A, L, across, each);
        return;
      }
    fwd_kernel<T, S, true><<<blocks, S::kLanes, 0, stream()>>>(A, L, across, each);
  });
}
template <class T, class S, bool ADD>
bool launch_bwd(const ScanArgs &A, const char *where) {
  return by_tiles<S>(A, where, [](const ScanArgs &A, unsigned blocks, const Look &L, uint32_t across, uint32_t each) {
    if constexpr (S::kTile < 256)
      if (L.tiles == 1) {
        bwd_kernel<T, S, ADD, false><<<blocks, S::kLanes, 0, stream()>>>(A, L, across, each);
        return;
      }
    bwd_kernel<T, S, ADD, true><<<blocks, S::kLanes, 0, stream()>>>(A, L, across, each);
  });
}
// Columns of 64 channels that a launch has, and the shapes of their tiles. A tile's lanes hold eight steps of four channels, so that
// a workgroup of 256 lanes takes 128 steps of 64 channels: with shorter tiles the slices are joined in less time and with longer
// ones states pass from tile to tile less often, which bounds a few long sequences. us, forward and backward of [batch, steps,
// channels], tiles of 64, 128 and 256 steps:
//   bf16 [1, 65536, 1024] 203 125 103, 251 200 207; [1, 65536, 256] 169 83 52, 175 90 65; [1, 32768, 2048] 135 100 97,
//   188 185 205; [1, 16384, 4096] 101 90 92, 164 170 201; [8, 4096, 1024] 52 48 53, 85 89 104; [32, 512, 2048] 47 49 49, 73 79 102
//   fp32 [1, 65536, 1024] 235 167 147, 326 268 287; [1, 16384, 4096] 153 142 143, 260 246 291; [8, 4096, 1024] 78 78 80,
//   139 138 151; [32, 512, 2048] 76 86 82, 140 153 152.
// The forward pass of fp32 over many columns is faster with twice the width, four steps a lane: [32, 512, 2048] 72,
// [8, 4096, 1024] 74, [5, 3001, 1003] 44 instead of 52, but [1, 16384, 4096] 151.
typedef Shape<16, 8, 64, 2> Short;
typedef Shape<16, 8, 128, 4> Middle;
typedef Shape<16, 8, 128, 2> MiddleBack;
typedef Shape<16, 8, 256, 4> Long;
typedef Shape<16, 8, 256, 2> LongBack;
typedef Shape<32, 4, 64, 5> Wide;
uint64_t columns_of(const ScanArgs &A) { return uint64_t(A.batch) * ceil_div(A.width, 64); }

// Operands that the last-level cache takes are read through it, others past the caches. Through / past, us: of the operands
// of the call before, forward and backward of [5, 3001, 1003] in fp32 106 / 134, forward of [32, 512, 2048] in bf16 37 / 43; forward of
// [1, 65536, 1024] 103 / 98, both of [8, 4096, 2048] 243 / 239.
constexpr uint64_t kCached = uint64_t(192) << 20;
template <class T>
bool past_caches(const ScanArgs &A, uint64_t operands) {
  return operands * A.batch * A.length * A.width * sizeof(T) > kCached;
}

template <class T>
bool launch_forward(ScanArgs A, const char *where) {
  A.past = past_caches<T>(A, 2);
  if (A.length <= kFewSteps) {
    const uint32_t quads = ceil_div(A.width, 4);
    few_kernel<T><<<ceil_div(uint64_t(A.batch) * quads, kFewLanes), kFewLanes, 0, stream()>>>(A, quads);
    return true;
  }
  const uint64_t columns = columns_of(A);
  if (columns <= 32 && A.length >= 8192) return launch_fwd<T, Long>(A, where);
  if constexpr (sizeof(T) == 4)
    if (A.length <= 64 * columns) return launch_fwd<T, Wide>(A, where);
  return launch_fwd<T, Middle>(A, where);
}
template <class T, bool ADD>
bool launch_backward(ScanArgs A, const char *where) {
  A.past = past_caches<T>(A, 3);
  const uint64_t columns = columns_of(A);
  if (columns <= 8 && A.length >= 8192) return launch_bwd<T, LongBack, ADD>(A, where);
  if (columns >= (sizeof(T) == 2 ? 64 : 512)) return launch_bwd<T, Short, ADD>(A, where);
  return launch_bwd<T, MiddleBack, ADD>(A, where);
}

}  // namespace
}  // namespace plast

using namespace plast;

extern "C" {

void plast_hip_set_recurrence_looks(int looks) { g_most_looks = looks > 0 ? uint32_t(looks) : 0; }

void gated_recurrence_hip_forward(const Tensor **inputs, Tensor *output, KernelParams params) {
  const char *where = "gated_recurrence_hip_forward";
  if (params.dim > 1) {
    report_error(where, "params.dim is 1 to keep the states for a backward pass and 0 not to, not %llu",
                 (unsigned long long)params.dim);
    return;
  }
  ScanArgs A;
  if (!scan_args(A, inputs, params.dim == 1, where)) return;
  if (!sequence(output, inputs[0]) || (numel(output) && overlapping(output))) {
    report_error(where, "the output must have f's type and shape, a contiguous last axis and steps that do not overlap");
    return;
  }
  if (!A.batch || !A.width) return;
  A.h = seq<char *>(output);
  if (A.length && (A.h.p == A.f.p || A.h.p == A.v.p)) {
    report_error(where, "the output lies in the place of f or v");
    return;
  }
  const Operand h("the output", output), last("the last state", inputs[4]), states("states", params.dim == 1 ? inputs[5] : nullptr),
      f("f", inputs[0]), v("v", inputs[1]), initial("the initial state", inputs[2]), lengths("lengths", inputs[3]);
  if (!apart(h, {&f, &v, &initial, &lengths, &last, &states}, where) || !apart(last, {&f, &v, &lengths, &states}, where) ||
      !apart(states, {&f, &v, &initial, &lengths}, where) || (A.last != A.initial && !apart(last, {&initial}, where)))
    return;
  if (!ensure_init()) return;
  bool ok = false;
  with_float_type(inputs[0]->dtype, [&](auto t) { ok = launch_forward<decltype(t)>(A, where); });
  if (ok) finish(where);
}

void gated_recurrence_hip_backward(Tensor **inputs, const Tensor *output, KernelParams params) {
  const char *where = "gated_recurrence_hip_backward";
  if (params.dim != 1) {
    report_error(where, "the backward pass needs the states that a forward pass with params.dim 1 has kept");
    return;
  }
  ScanArgs A;
  if (!scan_args(A, inputs, true, where)) return;
  const Tensor *f = inputs[0], *dy = output ? output->grad : nullptr, *dlast = inputs[4]->grad;
  if (dy) {
    if (!sequence(dy, f)) {
      report_error(where, "the output's gradient must have f's type and shape and a contiguous last axis");
      return;
    }
    A.dy = seq<const char *>(dy);
  }
  if (dlast) {
    if (!f32_vector(dlast, uint64_t(A.batch) * A.width)) {
      report_error(where, "the last state's gradient must be a contiguous FLOAT32 GPU tensor of its elements");
      return;
    }
    A.dlast = static_cast<const float *>(dlast->data);
  }
  Seq<char *> *const into[2] = {&A.df, &A.dv};
  for (int k = 0; k < 2; ++k) {
    if (!inputs[k]->requires_grad) continue;
    const Tensor *g = inputs[k]->grad;
    if (!sequence(g, f) || (numel(g) && overlapping(g))) {
      report_error(where, "the gradients of f and v must have their type and shape, a contiguous last axis and steps that do "
                   "not overlap");
      return;
    }
    *into[k] = seq<char *>(g);
  }
  if (A.df.p && A.df.p == A.dv.p) {
    report_error(where, "f and v have one gradient");
    return;
  }
  for (const char *g : {A.df.p, A.dv.p})
    if (g && A.length && (g == A.f.p || g == A.v.p || g == A.dy.p)) {
      report_error(where, "a gradient lies in the place of f, v or the output's gradient");
      return;
    }
  if (inputs[2]->requires_grad) {
    if (!f32_vector(inputs[2]->grad, uint64_t(A.batch) * A.width)) {
      report_error(where, "the initial state's gradient must be a contiguous FLOAT32 GPU tensor of its elements");
      return;
    }
    A.dinitial = static_cast<float *>(inputs[2]->grad->data);
    if (A.dinitial && A.dinitial == A.dlast) {
      report_error(where, "the initial and the last state have one gradient");
      return;
    }
  }
  const Operand to_f("the gradient of f", A.df.p ? inputs[0]->grad : nullptr), to_v("the gradient of v", A.dv.p ? inputs[1]->grad : nullptr),
      to_initial("the initial state's gradient", A.dinitial ? inputs[2]->grad : nullptr);
  const Operand at_f("f", f), v("v", inputs[1]), up("the output's gradient", dy), up_last("the last state's gradient", dlast),
      states("states", inputs[5]), lengths("lengths", inputs[3]);
  if (!apart(to_f, {&to_v, &to_initial}, where) || !apart(to_v, {&to_initial}, where)) return;
  for (const Operand *to : {&to_f, &to_v, &to_initial})
    if (!apart(*to, {&at_f, &v, &up, &up_last, &states, &lengths}, where)) return;
  if ((!A.df.p && !A.dv.p && !A.dinitial) || !A.batch || !A.width || !ensure_init()) return;
  bool ok = false;
  with_float_type(f->dtype, [&](auto t) {
    typedef decltype(t) T;
    ok = params.keepdim == 1 ? launch_backward<T, false>(A, where) : launch_backward<T, true>(A, where);
  });
  if (ok) finish(where);
}

}  // extern "C"
