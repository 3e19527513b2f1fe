// What the sources of the fused-ops extension share: 16-bit types, wave reductions, division by a
// number known at launch, and the host side's checks.
#pragma once
#include <hip/hip_runtime.h>
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <cstdint>
#include <cstring>

namespace {

typedef unsigned short u16;
template <int N>
using u16v = u16 __attribute__((ext_vector_type(N)));
typedef u16v<8> u16x8;

__device__ __forceinline__ float b2f(u16 v) { return __uint_as_float((unsigned)v << 16); }
__device__ __forceinline__ u16 f2b(float f) {
  __bf16 b = (__bf16)f;  // v_cvt_pk_bf16_f32: RNE, NaN stays NaN
  return __builtin_bit_cast(u16, b);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

inline hipStream_t stream() { return c10::hip::getCurrentHIPStream().stream(); }

#define LAUNCH_CHECK()                                                                         \
  do {                                                                                         \
    hipError_t e_ = hipGetLastError();                                                         \
    TORCH_CHECK(e_ == hipSuccess, "HIP launch failed: ", hipGetErrorString(e_));               \
  } while (0)

// What the operators without derivatives of derivatives refuse. A backward pass that is itself to be differentiated:
inline void no_second_order(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op, ": second derivatives are not implemented");
}
// A tangent of forward mode on any input: it needs no requires_grad, so that a call could pass the autograd node by,
// compute the value alone and lose the tangent without a word. Checked in front of all else.
template <typename... Tensors>
inline void no_tangents(const char* op, const Tensors&... inputs) {
  TORCH_CHECK(!(inputs._fw_grad(0).defined() || ...), op, ": forward-mode derivatives are not implemented");
}
inline at::Tensor or_none(const c10::optional<at::Tensor>& t) { return t ? *t : at::Tensor(); }

// ------------------------------------------------------------------------------ element types
// Storage of one element and its way to and from fp32 (round to nearest even).
struct BF16 {
  typedef u16 S;
  static constexpr at::ScalarType kType = at::kBFloat16;
  __device__ static __forceinline__ float get(u16 v) { return b2f(v); }
  __device__ static __forceinline__ u16 put(float f) { return f2b(f); }
};
struct FP16 {
  typedef u16 S;
  static constexpr at::ScalarType kType = at::kHalf;
  __device__ static __forceinline__ float get(u16 v) { return (float)__builtin_bit_cast(_Float16, v); }
  __device__ static __forceinline__ u16 put(float f) { return __builtin_bit_cast(u16, (_Float16)f); }
};
struct FP32 {
  typedef float S;
  static constexpr at::ScalarType kType = at::kFloat;
  __device__ static __forceinline__ float get(float v) { return v; }
  __device__ static __forceinline__ float put(float f) { return f; }
};

// N consecutive elements at any element address as one access (global memory takes wide accesses at
// any alignment of the element; aligned ones are the fast case).
template <typename S, int N>
struct alignas(sizeof(S)) Pack {
  S v[N];
};
template <typename S, int N>
__device__ __forceinline__ Pack<S, N> load_pack(const S* p) {
  typedef S vec __attribute__((ext_vector_type(N), aligned(sizeof(S))));
  Pack<S, N> r;
  if constexpr (N == 1) {
    r.v[0] = *p;
  } else {
    const vec x = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = x[i];
  }
  return r;
}
template <typename S, int N>
__device__ __forceinline__ void store_pack(S* p, const Pack<S, N>& r) {
  typedef S vec __attribute__((ext_vector_type(N), aligned(sizeof(S))));
  if constexpr (N == 1) {
    *p = r.v[0];
  } else {
    vec x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = r.v[i];
    *reinterpret_cast<vec*>(p) = x;
  }
}

// ------------------------------------------------------------------------------ division
// n / d for n < 2^31 and a divisor known at launch: multiply by the rounded-up reciprocal of d
// (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994).
struct FastDiv {
  unsigned d, m, s;
  FastDiv() : d(1), m(1), s(0) {}
  explicit FastDiv(unsigned div) : d(div), s(0) {
    while (s < 31 && (1u << s) < div) ++s;
    m = (unsigned)(((1ull << 32) * ((1ull << s) - div)) / div + 1);
  }
  __device__ __forceinline__ unsigned div(unsigned n) const { return (__umulhi(n, m) + n) >> s; }
  __device__ __forceinline__ unsigned divmod(unsigned n, unsigned& rem) const {
    const unsigned q = div(n);
    rem = n - q * d;
    return q;
  }
};

}  // namespace
