// gated_recurrence.hip — the gated linear recurrence along a sequence, each channel by itself, and its gradients:
//   a = sigmoid(f),  z = 1 - a,  h[t] = a[t] h[t-1] + z[t] v[t],
//   dh[t] = dy[t] + a[t+1] dh[t+1],  dv = z dh,  df = dh (h[t-1] - v) a z,  dh[-1] = a[0] dh[0].
//
// With e = exp(-|f|), the larger of a and z is 1 / (1 + e) and the smaller e / (1 + e), each to some 1e-7 of itself: next to 1
// the larger has lost what the smaller holds. A step multiplies the state by a, whose rounding would add up over a long memory
// if steps were all there is: so runs of eight steps are short cuts of their own, which take what they do to a state from the
// smaller sides where those count (Share), and every run starts from there.
// A product with a factor of 0 is 0 whatever the other factor is (v_mul_legacy_f32): a gate so far out that one side is 0
// selects, and lets no NaN through.
#include <cfloat>
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
};

extern "C" __device__ float mul_legacy(float, float) __asm("llvm.amdgcn.fmul.legacy");

// Both sides of a gate.
struct Gate {
  float a, z;
  __device__ __forceinline__ explicit Gate(float f) {
    const float e = __builtin_amdgcn_exp2f(-1.44269504f * fabsf(f));
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
    return shut ? -0.0f : c < 0.9375f ? c : -fmaxf(a, FLT_MIN);
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
    *reinterpret_cast<typename Quad<T>::any *>(p) = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < n) p[e] = v[e];
}
// The same at a lane's offset in bytes from a step's address, which is the same for all lanes.
template <class T>
__device__ __forceinline__ typename Quad<T>::vec load_at(const void *step, uint32_t offset, int n, float otherwise = 0.0f) {
  return load_quad(reinterpret_cast<const T *>(static_cast<const char *>(step) + offset), n, otherwise);
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

// A tile is a chunk of kChunk steps of 64 channels: 16 lanes across, four channels each, and slices of some steps, a slice a
// lane's. Every lane finds its slice's share and what it adds from a state of 0, the slices' are joined in LDS, and each lane goes
// through its steps again from the state that its slice starts with. The forward pass has 16 slices of eight steps; the
// backward pass, which holds twice as much of a step, 32 of four.
constexpr uint32_t kLanes = 256, kAcross = 16, kTileWidth = 4 * kAcross;
constexpr uint32_t kFwdSlices = 16, kBwdSlices = 32;

// What tiles of one column of tiles leave for those behind them: `plus` and `code` of the chunk alone, and the state after it.
// A word's upper half says that it is there, so each word counts by itself.
struct Record {
  uint64_t code[kTileWidth], plus[kTileWidth], state[kTileWidth];
};
struct Look {
  uint32_t *ticket;
  Record *records;  // [chunks][batch, columns]
};
__device__ __forceinline__ void put_word(uint64_t *p, float v) { put_shared(p, uint64_t(1) << 32 | __float_as_uint(v)); }
__device__ __forceinline__ bool is_there(uint64_t w) { return (w >> 32) != 0; }
__device__ __forceinline__ float word_value(uint64_t w) { return __uint_as_float(uint32_t(w)); }

__global__ __launch_bounds__(kLanes) void clear_kernel(uint64_t *p, uint64_t n) {
  const uint64_t i = uint64_t(blockIdx.x) * kLanes + threadIdx.x;
  if (i < n) p[i] = 0;
}

// The state that a tile starts with, by one wave, a lane a channel: of the `n` tiles before it (`step` records apart) the
// nearest whose state is there is found, and the shares of those between are applied to it one after the other, as they
// themselves do: the bits do not depend on which it was.
// Tiles take tickets in the order of their chunks, so those before are at work or done, and each leaves its own share before it
// waits for anything: every wait ends. kMostLooks, some seconds, bounds it all the same; the state is NaN then.
constexpr uint32_t kMostLooks = 1u << 22, kWindow = 4;
__device__ __forceinline__ float look_back(Record *mine, int64_t step, uint32_t n, uint32_t lane, uint64_t ready, float code,
                                           float plus) {
  if (__all(is_there(ready))) return word_value(ready);
  put_word(&mine->code[lane], code);
  put_word(&mine->plus[lane], plus);
  uint32_t d0 = 1, looks = 0;  // the nearest tile of a window is d0 before this one
  for (;;) {
    uint64_t s[kWindow], c[kWindow], p[kWindow];
#pragma unroll
    for (uint32_t w = 0; w < kWindow; ++w) {
      const Record *r = mine - step * int64_t(d0 + w < n ? d0 + w : n);
      s[w] = get_shared(&r->state[lane]);
      c[w] = get_shared(&r->code[lane]);
      p[w] = get_shared(&r->plus[lane]);
    }
    uint32_t at = 0;  // tiles of the window whose shares are there and states are not
    bool found = false, whole = true;
    float x = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < kWindow; ++w)
      if (!found && whole) {
        found = __all(is_there(s[w]));
        if (found) x = word_value(s[w]);
        else if (__all(is_there(c[w]) && is_there(p[w]))) ++at;
        else whole = false;
      }
    if (found) {
#pragma unroll
      for (uint32_t w = kWindow; w-- > 0;)
        if (w < at) x = apply(word_value(c[w]), word_value(p[w]), x);
      for (uint32_t d = d0; d > 1;) {  // the windows before, which are there
        d -= kWindow;
#pragma unroll
        for (uint32_t w = 0; w < kWindow; ++w) {
          const Record *r = mine - step * int64_t(d + w);
          c[w] = get_shared(&r->code[lane]);
          p[w] = get_shared(&r->plus[lane]);
        }
#pragma unroll
        for (uint32_t w = kWindow; w-- > 0;) x = apply(word_value(c[w]), word_value(p[w]), x);
      }
      return x;
    }
    if (whole) d0 += kWindow;
    else if (++looks == kMostLooks) return __builtin_nanf("");
    else __builtin_amdgcn_s_sleep(1);
  }
}

struct TileAt {
  uint32_t chunk, b, column;
};
// Where a tile lies in a sequence operand: the address of its step k, and the offset from there of a lane whose slice starts
// `first` steps into the tile.
template <class T, class P>
struct TileSeq {
  P p;
  int64_t step;
  uint32_t offset;
  __device__ __forceinline__ TileSeq(const Seq<P> &s, const TileAt &at, uint32_t first, uint32_t across) {
    p = s.p + (int64_t(at.b) * s.b + int64_t(at.chunk * kChunk) * s.t + at.column * kTileWidth) * int64_t(sizeof(T));
    step = s.t * int64_t(sizeof(T));
    offset = (first * uint32_t(s.t) + 4 * across) * uint32_t(sizeof(T));
  }
  __device__ __forceinline__ P at(uint32_t k) const { return p + step * k; }
};
__device__ __forceinline__ TileAt tile_at(const ScanArgs &A, uint32_t i, uint32_t columns) {
  const uint32_t row = A.batch * columns, chunk = i / row, rest = i - chunk * row, b = rest / columns;
  return {chunk, b, rest - b * columns};
}

template <class T, bool MANY>
__global__ __launch_bounds__(kAcross * kFwdSlices, 3) void fwd_kernel(ScanArgs A, Look K, uint32_t columns) {
  constexpr uint32_t kSlices = kFwdSlices, kSteps = kChunk / kSlices;
  __shared__ __align__(16) float codes[kSlices][kTileWidth], plus[kSlices][kTileWidth];
  __shared__ uint32_t taken;
  uint32_t tile = blockIdx.x;
  if constexpr (MANY) {
    if (threadIdx.x == 0) taken = atomicAdd(K.ticket, 1u);
    __syncthreads();
    tile = __builtin_amdgcn_readfirstlane(taken);
  }
  const TileAt at = tile_at(A, tile, columns);
  const uint32_t end = live_steps(A, at.b), across = threadIdx.x & (kAcross - 1), slice = threadIdx.x / kAcross;
  const uint32_t c = at.column * kTileWidth + 4 * across, t0 = at.chunk * kChunk + slice * kSteps;
  const int n = int(A.width) - int(c);
  const TileSeq<T, char *> y(A.h, at, slice * kSteps, across);
  if (at.chunk > 0 && at.chunk * kChunk >= end) {  // padding alone
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k)
      if (t0 + k < A.length) store_at<T>(y.at(k), y.offset, f4(0.0f), n);
    return;
  }
  const TileSeq<T, const char *> f(A.f, at, slice * kSteps, across), v(A.v, at, slice * kSteps, across);
  typename Quad<T>::vec gates[kSteps], val[kSteps];
  // a tile of channels and steps that are all there takes no bounds
  const bool whole = (at.column + 1) * kTileWidth <= A.width && (at.chunk + 1) * kChunk <= end;
  if (whole) {
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      gates[k] = load_at<T>(f.at(k), f.offset, 4);
      val[k] = load_at<T>(v.at(k), v.offset, 4);
    }
  } else {
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      const int m = t0 + k < end ? n : 0;
      gates[k] = load_at<T>(f.at(k), f.offset, m, kHold);
      val[k] = load_at<T>(v.at(k), v.offset, m);
    }
  }
  // wave 0's lanes are the tile's channels while the slices are joined
  const uint32_t lane = threadIdx.x, channel = at.column * kTileWidth + lane;
  const bool joins = threadIdx.x < 64, inside = channel < A.width;
  Record *mine = nullptr;
  uint64_t ready = 0;
  float start = 0.0f;
  if (joins) {
    if (MANY && at.chunk > 0) {
      mine = K.records + tile;
      ready = get_shared(&(mine - A.batch * columns)->state[lane]);
    } else if (inside) {
      if constexpr (MANY) mine = K.records + tile;
      start = A.initial[uint64_t(at.b) * A.width + channel];
    }
  }
  f4 keep[kSteps], add[kSteps], sum = 0.0f;
  Share share[4];
#pragma unroll
  for (uint32_t k = 0; k < kSteps; ++k) {
    const f4 x = to_f4<T>(gates[k]), u = to_f4<T>(val[k]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const Gate g(x[e]);
      keep[k][e] = g.a;
      add[k][e] = mul_legacy(g.z, u[e]);
      share[e].step(g.a, g.z);
      sum[e] = mul_legacy(g.a, sum[e]) + add[k][e];
    }
  }
  f4 code;
#pragma unroll
  for (int e = 0; e < 4; ++e) code[e] = share[e].code();
  *reinterpret_cast<f4 *>(&codes[slice][4 * across]) = code;
  *reinterpret_cast<f4 *>(&plus[slice][4 * across]) = sum;
  __syncthreads();
  if (joins) {
    float cs[kSlices], ps[kSlices];
#pragma unroll
    for (uint32_t i = 0; i < kSlices; ++i) cs[i] = codes[i][lane], ps[i] = plus[i][lane];
    if constexpr (MANY) {
      Share joined;
      float all = 0.0f;
#pragma unroll
      for (uint32_t i = 0; i < kSlices; ++i) joined.join(cs[i]), all = apply(cs[i], ps[i], all);
      if (at.chunk > 0) start = look_back(mine, int64_t(A.batch) * columns, at.chunk, lane, ready, joined.code(), all);
      put_word(&(K.records + tile)->state[lane], apply(joined.code(), all, start));
    }
    if (A.states && inside) A.states[(uint64_t(at.b) * A.chunks + at.chunk) * A.width + channel] = start;
    if (end == 0 && inside) A.last[uint64_t(at.b) * A.width + channel] = start;
#pragma unroll
    for (uint32_t i = 0; i < kSlices; ++i) {
      plus[i][lane] = start;
      start = apply(cs[i], ps[i], start);
    }
  }
  __syncthreads();
  f4 h = *reinterpret_cast<const f4 *>(&plus[slice][4 * across]);
  if (whole) {
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = mul_legacy(keep[k][e], h[e]) + add[k][e];
      store_at<T>(y.at(k), y.offset, h, 4);
    }
    if (t0 + kSteps == end) store_quad<float>(A.last + uint64_t(at.b) * A.width + c, h, 4);
    return;
  }
#pragma unroll
  for (uint32_t k = 0; k < kSteps; ++k) {
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = mul_legacy(keep[k][e], h[e]) + add[k][e];
    if (t0 + k < A.length) store_at<T>(y.at(k), y.offset, t0 + k < end ? h : f4(0.0f), n);
    if (t0 + k + 1 == end) store_quad<float>(A.last + uint64_t(at.b) * A.width + c, h, n);
  }
}

template <class T, bool ADD>
__device__ __forceinline__ void put_at(char *step, uint32_t offset, f4 f, int n) {
  if constexpr (ADD) f += to_f4<T>(load_at<T>(step, offset, n));
  store_at<T>(step, offset, f, n);
}

template <class T, bool ADD, bool MANY>
__global__ __launch_bounds__(kAcross * kBwdSlices, 4) void bwd_kernel(ScanArgs A, Look K, uint32_t columns) {
  constexpr uint32_t kSlices = kBwdSlices, kSteps = kChunk / kSlices;
  __shared__ __align__(16) float codes[kSlices][kTileWidth], plus[kSlices][kTileWidth], back[kSlices][kTileWidth];
  __shared__ uint32_t taken;
  uint32_t tile = blockIdx.x;
  if constexpr (MANY) {
    if (threadIdx.x == 0) taken = atomicAdd(K.ticket, 1u);
    __syncthreads();
    tile = __builtin_amdgcn_readfirstlane(taken);
  }
  TileAt at = tile_at(A, tile, columns);
  at.chunk = A.chunks - 1 - at.chunk;
  const uint32_t end = live_steps(A, at.b), across = threadIdx.x & (kAcross - 1), slice = threadIdx.x / kAcross;
  const uint32_t c = at.column * kTileWidth + 4 * across, t0 = at.chunk * kChunk + slice * kSteps;
  const int n = int(A.width) - int(c);
  const TileSeq<T, char *> df(A.df, at, slice * kSteps, across), dv(A.dv, at, slice * kSteps, across);
  if (at.chunk > 0 && at.chunk * kChunk >= end) {  // padding alone
    if (!ADD)
#pragma unroll
      for (uint32_t k = 0; k < kSteps; ++k)
        if (t0 + k < A.length) {
          if (A.df.p) store_at<T>(df.at(k), df.offset, f4(0.0f), n);
          if (A.dv.p) store_at<T>(dv.at(k), dv.offset, f4(0.0f), n);
        }
    return;
  }
  const TileSeq<T, const char *> f(A.f, at, slice * kSteps, across), v(A.v, at, slice * kSteps, across), dy(A.dy, at, slice * kSteps, across);
  typename Quad<T>::vec gates[kSteps], val[kSteps], up[kSteps];
  const bool whole = (at.column + 1) * kTileWidth <= A.width && (at.chunk + 1) * kChunk <= end && A.dy.p && A.df.p && A.dv.p;
  if (whole) {
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      gates[k] = load_at<T>(f.at(k), f.offset, 4);
      val[k] = load_at<T>(v.at(k), v.offset, 4);
      up[k] = load_at<T>(dy.at(k), dy.offset, 4);
    }
  } else {
#pragma unroll
    for (uint32_t k = 0; k < kSteps; ++k) {
      const int m = t0 + k < end ? n : 0;
      gates[k] = load_at<T>(f.at(k), f.offset, m, kHold);
      val[k] = load_at<T>(v.at(k), v.offset, m);
      up[k] = load_at<T>(dy.at(k), dy.offset, A.dy.p ? m : 0);
    }
  }
  // waves 0 and 1 join the slices, one forward and one from the end
  const uint32_t lane = threadIdx.x & 63, channel = at.column * kTileWidth + lane, wave = threadIdx.x / 64;
  const bool inside = channel < A.width, last = at.chunk * kChunk + kChunk >= end;  // last: nothing comes from behind
  const uint64_t state_at = uint64_t(at.b) * A.width + channel;
  float start = 0.0f;
  uint64_t ready = 0;
  if (wave == 0 && inside && end) start = A.states[(uint64_t(at.b) * A.chunks + at.chunk) * A.width + channel];
  if (MANY && wave == 1 && !last) ready = get_shared(&(K.records + tile - A.batch * columns)->state[lane]);
  f4 dlast = 0.0f;
  if (A.dlast && end && t0 < end && end <= t0 + kSteps) dlast = load_quad<float>(A.dlast + uint64_t(at.b) * A.width + c, n);
  f4 keep[kSteps], into[kSteps], sum = 0.0f, rev = 0.0f;
  Share share[4];
#pragma unroll
  for (uint32_t k = 0; k < kSteps; ++k) {
    const f4 x = to_f4<T>(gates[k]), u = to_f4<T>(val[k]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const Gate g(x[e]);
      keep[k][e] = g.a;
      into[k][e] = g.z;
      share[e].step(g.a, g.z);
      sum[e] = mul_legacy(g.a, sum[e]) + mul_legacy(g.z, u[e]);
    }
  }
#pragma unroll
  for (uint32_t k = kSteps; k-- > 0;) {
    f4 d = to_f4<T>(up[k]);
    if (t0 + k + 1 == end) d += dlast;
#pragma unroll
    for (int e = 0; e < 4; ++e) rev[e] = mul_legacy(keep[k][e], rev[e] + d[e]);
  }
  f4 code;
#pragma unroll
  for (int e = 0; e < 4; ++e) code[e] = share[e].code();
  *reinterpret_cast<f4 *>(&codes[slice][4 * across]) = code;
  *reinterpret_cast<f4 *>(&plus[slice][4 * across]) = sum;
  *reinterpret_cast<f4 *>(&back[slice][4 * across]) = rev;
  __syncthreads();
  keep_raw(val);
  keep_raw(up);
  if (wave == 0) {
#pragma unroll 8
    for (uint32_t i = 0; i < kSlices; ++i) {
      const float after = apply(codes[i][lane], plus[i][lane], start);
      plus[i][lane] = start;
      start = after;
    }
  } else if (wave == 1) {
    float from = 0.0f;  // a dh of the step behind the tile
    if constexpr (MANY) {
      Share joined;
      float all = 0.0f;
#pragma unroll 8
      for (uint32_t i = kSlices; i-- > 0;) joined.join(codes[i][lane]), all = apply(codes[i][lane], back[i][lane], all);
      if (!last)
        from = look_back(K.records + tile, int64_t(A.batch) * columns, A.chunks - 1 - at.chunk, lane, ready, joined.code(), all);
      put_word(&(K.records + tile)->state[lane], apply(joined.code(), all, from));
    }
#pragma unroll 8
    for (uint32_t i = kSlices; i-- > 0;) {
      const float after = apply(codes[i][lane], back[i][lane], from);
      back[i][lane] = from;
      from = after;
    }
    if (at.chunk == 0 && A.dinitial && inside) {
      if (end == 0 && A.dlast) from = A.dlast[state_at];
      A.dinitial[state_at] = ADD ? A.dinitial[state_at] + from : from;
    }
  }
  __syncthreads();
  f4 h = *reinterpret_cast<const f4 *>(&plus[slice][4 * across]);
  f4 d = *reinterpret_cast<const f4 *>(&back[slice][4 * across]);
  f4 dh[kSteps];
  keep_raw(up);
  keep_raw(val);
#pragma unroll
  for (uint32_t k = kSteps; k-- > 0;) {
    dh[k] = d + to_f4<T>(up[k]);
    if (t0 + k + 1 == end) dh[k] += dlast;
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
    if (t0 + k >= end) to_f = to_v = f4(0.0f);
    if (t0 + k < (ADD ? end : A.length)) {
      if (A.df.p) put_at<T, ADD>(df.at(k), df.offset, to_f, n);
      if (A.dv.p) put_at<T, ADD>(dv.at(k), dv.offset, to_v, n);
    }
  }
}

// ------------------------------------------------------------------------- few steps

// A lane four channels, step by step: tokens of a decode batch.
constexpr uint32_t kFewSteps = 16;
template <class T>
__global__ __launch_bounds__(kLanes) void few_kernel(ScanArgs A, uint32_t quads) {
  const uint64_t i = uint64_t(blockIdx.x) * kLanes + threadIdx.x;
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
        const Gate g(x[e]);
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
  return t && (t->ndim != 3 || t->shape[1] <= 1 || t->strides[1] <= kMostStep) && t->device == GPU && t->dtype == f->dtype && same_shape(t, f) && (numel(f) == 0 || t->data) &&
         (f->shape[2] <= 1 || t->strides[2] == 1);
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

// Clears the records and the ticket of a launch over several chunks.
bool look_at(Look &K, uint64_t tiles, const char *where) {
  const uint64_t words = 32 + tiles * sizeof(Record) / 8;  // the ticket has 256 bytes
  uint64_t *p = static_cast<uint64_t *>(partials(words * 8, where));
  if (!p) return false;
  K.ticket = reinterpret_cast<uint32_t *>(p);
  K.records = reinterpret_cast<Record *>(p + 32);
  clear_kernel<<<ceil_div(words, kLanes), kLanes, 0, stream()>>>(p, words);
  return true;
}
// launch(columns, tiles, records, whether there are several chunks)
template <class F>
bool by_tiles(const ScanArgs &A, const char *where, F &&launch) {
  const uint32_t columns = ceil_div(A.width, kTileWidth);
  const uint64_t tiles = uint64_t(A.batch) * columns * A.chunks;
  if (tiles > max_blocks(kAcross * kBwdSlices)) {
    report_error(where, "%llu chunks of 64 channels are not supported", (unsigned long long)tiles);
    return false;
  }
  Look K{nullptr, nullptr};
  if (A.chunks > 1 && !look_at(K, tiles, where)) return false;
  launch(columns, unsigned(tiles), K, A.chunks > 1);
  return true;
}

template <class T>
bool launch_forward(const ScanArgs &A, const char *where) {
  if (A.length <= kFewSteps) {
    const uint32_t quads = ceil_div(A.width, 4);
    few_kernel<T><<<ceil_div(uint64_t(A.batch) * quads, kLanes), kLanes, 0, stream()>>>(A, quads);
    return true;
  }
  return by_tiles(A, where, [&](uint32_t columns, unsigned tiles, const Look &K, bool many) {
    if (many) fwd_kernel<T, true><<<tiles, kAcross * kFwdSlices, 0, stream()>>>(A, K, columns);
    else fwd_kernel<T, false><<<tiles, kAcross * kFwdSlices, 0, stream()>>>(A, K, columns);
  });
}
template <class T, bool ADD>
bool launch_backward(ScanArgs A, const char *where) {
  if (A.length == 0) A.chunks = 1;  // what comes for the last state is the initial one's
  return by_tiles(A, where, [&](uint32_t columns, unsigned tiles, const Look &K, bool many) {
    if (many) bwd_kernel<T, ADD, true><<<tiles, kAcross * kBwdSlices, 0, stream()>>>(A, K, columns);
    else bwd_kernel<T, ADD, false><<<tiles, kAcross * kBwdSlices, 0, stream()>>>(A, K, columns);
  });
}

}  // namespace
}  // namespace plast

using namespace plast;

extern "C" {

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
  if (!A.batch || !A.width || !ensure_init()) return;
  A.h = seq<char *>(output);
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
  if (inputs[2]->requires_grad) {
    if (!f32_vector(inputs[2]->grad, uint64_t(A.batch) * A.width)) {
      report_error(where, "the initial state's gradient must be a contiguous FLOAT32 GPU tensor of its elements");
      return;
    }
    A.dinitial = static_cast<float *>(inputs[2]->grad->data);
  }
  if ((!A.df.p && !A.dv.p && !A.dinitial) || !A.batch || !A.width || !ensure_init()) return;
  bool ok = false;
  with_float_type(f->dtype, [&](auto t) {
    typedef decltype(t) T;
    ok = params.keepdim == 1 ? launch_backward<T, false>(A, where) : launch_backward<T, true>(A, where);
  });
  if (ok) finish(where);
}

}  // extern "C"
