// What the model operators' kernels (embedding.hip, qk_rope.hip, distill.hip) share: element types, accesses of 2 to 16
// bytes, reductions over a wave of 64 lanes, and the launch helpers of their host side.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <limits>
#include <string>

#include "common.h"

namespace tandem_hip {
namespace ops {

constexpr int kWave = 64;

// 16-bit floats convert in hardware (bf16: v_cvt_pk_bf16_f32), once, to nearest even; a NaN stays a NaN.
template <typename T>
__device__ __forceinline__ float widen(T x) { return static_cast<float>(x); }
template <typename T>
__device__ __forceinline__ T narrow(float x) { return static_cast<T>(x); }

// kBytes bytes of elements: one access of that width.
template <int kBytes> struct RawOf;
template <> struct RawOf<16> { typedef uint32_t type __attribute__((ext_vector_type(4))); };
template <> struct RawOf<8> { typedef uint32_t type __attribute__((ext_vector_type(2))); };
template <> struct RawOf<4> { typedef uint32_t type; };
template <> struct RawOf<2> { typedef uint16_t type; };

template <typename T, int kN>
struct Pack {
  using raw_t = typename RawOf<kN * static_cast<int>(sizeof(T))>::type;
  T v[kN];
  static __device__ __forceinline__ Pack of(raw_t raw) {
    Pack p;
    __builtin_memcpy(&p, &raw, sizeof(raw));
    return p;
  }
  static __device__ __forceinline__ Pack load(const T* at) { return of(*reinterpret_cast<const raw_t*>(at)); }
  static __device__ __forceinline__ Pack load_nt(const T* at) { return of(__builtin_nontemporal_load(reinterpret_cast<const raw_t*>(at))); }
  __device__ __forceinline__ raw_t raw() const {
    raw_t r;
    __builtin_memcpy(&r, this, sizeof(r));
    return r;
  }
  __device__ __forceinline__ void store(T* at) const { *reinterpret_cast<raw_t*>(at) = raw(); }
  __device__ __forceinline__ void store_nt(T* at) const { __builtin_nontemporal_store(raw(), reinterpret_cast<raw_t*>(at)); }
};

// ---- host side

// The widest access, in bytes (16 at most, `least` at least), that divides every one of the addresses and pitches or-ed into `bits`.
inline int access_width(uintptr_t bits, int least) {
  int w = 16;
  while (w > least && bits % static_cast<uintptr_t>(w) != 0) w /= 2;
  return w;
}

inline void check_launch(const char* what) { check_hip(hipGetLastError(), what); }

inline void require(bool ok, const char* message) {
  if (!ok) throw Invalid(message);
}

inline bool operator_dtype(int dtype) { return dtype == TDM_F32 || dtype == TDM_F16 || dtype == TDM_BF16; }

// Calls f with a value of the element type that `dtype` names.
template <class F>
void with_dtype(int dtype, F&& f) {
  switch (dtype) {
    case TDM_F32: f(float{}); return;
    case TDM_F16: f(_Float16{}); return;
    case TDM_BF16: f(__bf16{}); return;
    default: throw Invalid("the dtype must be float32, float16 or bfloat16");
  }
}

}  // namespace ops
}  // namespace tandem_hip
