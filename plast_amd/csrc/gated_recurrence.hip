// gated_recurrence.hip — the gated linear recurrence along a sequence, each channel by itself, and its gradients:
//   a = sigmoid(f),  z = 1 - a,  h[t] = a[t] h[t-1] + z[t] v[t],
//   dh[t] = dy[t] + a[t+1] dh[t+1],  dv = z dh,  df = dh (h[t-1] - v) a z,  dh[-1] = a[0] dh[0].
//
// A gate that remembers for long has an a next to 1, whose fp32 value has lost the digits of z that say for how long. So a
// gate is held as its smaller side, s = min(a, z) = e / (1 + e) with e = exp(-|f|), which is exact to some 1e-7 of itself at
// either end, and as which side that is:
//   h' = f > 0 ? h + s (v - h) : v + s (h - v).
// A gate so far out that s is 0 selects: h' is h or v whatever the other holds, NaN too.
#include <cfloat>
#include <cmath>
#include <cstring>
#include <type_traits>

#include "rows.hpp"

namespace plast {
namespace {

constexpr uint32_t kChunk = PLAST_RECURRENCE_CHUNK;
constexpr int kBlock256 = 256;

// A sequence operand: strides of the batch and of time, in elements.
template <class P>
struct Seq {
  P p;
  int64_t b, t;
};
struct ScanArgs {
  Seq<const void *> f, v, dy;
  Seq<void *> h, df, dv;
  const float *initial, *dlast;
  const int32_t *lengths;
  float *last, *states, *dinitial;
  uint32_t batch, length, width, chunks;
};

// The smaller side of a gate, and whether the state is what it mostly keeps.
struct Gate {
  float s;
  bool keep;
  __device__ __forceinline__ explicit Gate(float f) {
    const float e = __builtin_amdgcn_exp2f(-1.44269504f * fabsf(f));
    s = e / (1.0f + e);
    keep = f > 0.0f;
  }
  __device__ __forceinline__ float next(float h, float v) const {
    const float base = keep ? h : v, other = keep ? v : h;
    return s == 0.0f ? base : __builtin_fmaf(s, other - base, base);
  }
  // z x and a x
  __device__ __forceinline__ float take(float x) const { return side(x, !keep); }
  __device__ __forceinline__ float hold(float x) const { return side(x, keep); }
  __device__ __forceinline__ float side(float x, bool larger) const {
    if (s == 0.0f) return larger ? x : 0.0f;
    return larger ? __builtin_fmaf(-s, x, x) : s * x;
  }
  // d next / d f for upstream dh
  __device__ __forceinline__ float slope(float dh, float h, float v) const {
    return s == 0.0f ? 0.0f : dh * (h - v) * __builtin_fmaf(-s, s, s);
  }
};

__device__ __forceinline__ uint32_t live_steps(const ScanArgs &A, uint32_t b) {
  const int32_t n = A.lengths[b];
  return n < 0 ? 0 : uint32_t(n) < A.length ? uint32_t(n) : A.length;
}

// A lane a channel, step by step.
template <class T>
__global__ __launch_bounds__(kBlock256) void fwd_kernel(ScanArgs A) {
  const uint64_t i = uint64_t(blockIdx.x) * kBlock256 + threadIdx.x;
  if (i >= uint64_t(A.batch) * A.width) return;
  const uint32_t b = uint32_t(i / A.width), c = uint32_t(i - uint64_t(b) * A.width), end = live_steps(A, b);
  const T *f = static_cast<const T *>(A.f.p) + int64_t(b) * A.f.b + c;
  const T *v = static_cast<const T *>(A.v.p) + int64_t(b) * A.v.b + c;
  T *y = static_cast<T *>(A.h.p) + int64_t(b) * A.h.b + c;
  float h = A.initial[i];
  for (uint32_t t = 0; t < A.length; ++t) {
    if (A.states && t % kChunk == 0) A.states[(uint64_t(b) * A.chunks + t / kChunk) * A.width + c] = h;
    if (t < end) h = Gate(float(f[int64_t(t) * A.f.t])).next(h, float(v[int64_t(t) * A.v.t]));
    y[int64_t(t) * A.h.t] = T(t < end ? h : 0.0f);
  }
  A.last[i] = h;
}

template <class T, bool ADD>
__device__ __forceinline__ void put(T *p, float v) {
  *p = T(ADD ? float(*p) + v : v);
}

template <class T, bool ADD>
__global__ __launch_bounds__(kBlock256) void bwd_kernel(ScanArgs A) {
  const uint64_t i = uint64_t(blockIdx.x) * kBlock256 + threadIdx.x;
  if (i >= uint64_t(A.batch) * A.width) return;
  const uint32_t b = uint32_t(i / A.width), c = uint32_t(i - uint64_t(b) * A.width), end = live_steps(A, b);
  const T *f = static_cast<const T *>(A.f.p) + int64_t(b) * A.f.b + c;
  const T *v = static_cast<const T *>(A.v.p) + int64_t(b) * A.v.b + c;
  const T *dy = A.dy.p ? static_cast<const T *>(A.dy.p) + int64_t(b) * A.dy.b + c : nullptr;
  T *df = A.df.p ? static_cast<T *>(A.df.p) + int64_t(b) * A.df.b + c : nullptr;
  T *dv = A.dv.p ? static_cast<T *>(A.dv.p) + int64_t(b) * A.dv.b + c : nullptr;
  float g = A.dlast ? A.dlast[i] : 0.0f;
  float before[kChunk];
  for (uint32_t t = A.length; t-- > 0;) {
    if (t >= end) {
      if (df) put<T, ADD>(df + int64_t(t) * A.df.t, 0.0f);
      if (dv) put<T, ADD>(dv + int64_t(t) * A.dv.t, 0.0f);
      continue;
    }
    const uint32_t t0 = t / kChunk * kChunk;
    if (t == end - 1 || t == t0 + kChunk - 1) {
      float h = A.states[(uint64_t(b) * A.chunks + t / kChunk) * A.width + c];
      for (uint32_t k = t0; k <= t; ++k) {
        before[k - t0] = h;
        h = Gate(float(f[int64_t(k) * A.f.t])).next(h, float(v[int64_t(k) * A.v.t]));
      }
    }
    const Gate gate{float(f[int64_t(t) * A.f.t])};
    const float dh = (dy ? float(dy[int64_t(t) * A.dy.t]) : 0.0f) + g;
    if (dv) put<T, ADD>(dv + int64_t(t) * A.dv.t, gate.take(dh));
    if (df) put<T, ADD>(df + int64_t(t) * A.df.t, gate.slope(dh, before[t - t0], float(v[int64_t(t) * A.v.t])));
    g = gate.hold(dh);
  }
  if (A.dinitial) put<float, ADD>(A.dinitial + i, g);
}

// ------------------------------------------------------------------------- host

bool sequence(const Tensor *t, const Tensor *f) {
  return t && t->device == GPU && t->dtype == f->dtype && same_shape(t, f) && (numel(f) == 0 || t->data) &&
         (f->shape[2] <= 1 || t->strides[2] == 1);
}
template <class P>
Seq<P> seq(const Tensor *t) {
  return {t->data, t->shape[0] > 1 ? int64_t(t->strides[0]) : 0, t->shape[1] > 1 ? int64_t(t->strides[1]) : 0};
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
  A.f = seq<const void *>(f);
  A.v = seq<const void *>(v);
  A.initial = static_cast<const float *>(initial->data);
  A.lengths = static_cast<const int32_t *>(lengths->data);
  A.last = static_cast<float *>(last->data);
  A.batch = uint32_t(B);
  A.length = uint32_t(L);
  A.width = uint32_t(D);
  return true;
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
  A.h = seq<void *>(output);
  with_float_type(inputs[0]->dtype, [&](auto t) {
    fwd_kernel<decltype(t)><<<ceil_div(uint64_t(A.batch) * A.width, kBlock256), kBlock256, 0, stream()>>>(A);
  });
  finish(where);
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
    A.dy = seq<const void *>(dy);
  }
  if (dlast) {
    if (!f32_vector(dlast, uint64_t(A.batch) * A.width)) {
      report_error(where, "the last state's gradient must be a contiguous FLOAT32 GPU tensor of its elements");
      return;
    }
    A.dlast = static_cast<const float *>(dlast->data);
  }
  Seq<void *> *const into[2] = {&A.df, &A.dv};
  for (int k = 0; k < 2; ++k) {
    if (!inputs[k]->requires_grad) continue;
    const Tensor *g = inputs[k]->grad;
    if (!sequence(g, f) || (numel(g) && overlapping(g))) {
      report_error(where, "the gradients of f and v must have their type and shape, a contiguous last axis and steps that do "
                   "not overlap");
      return;
    }
    *into[k] = seq<void *>(g);
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
  const unsigned blocks = ceil_div(uint64_t(A.batch) * A.width, kBlock256);
  with_float_type(f->dtype, [&](auto t) {
    typedef decltype(t) T;
    if (params.keepdim == 1) bwd_kernel<T, false><<<blocks, kBlock256, 0, stream()>>>(A);
    else bwd_kernel<T, true><<<blocks, kBlock256, 0, stream()>>>(A);
  });
  finish(where);
}

}  // extern "C"
