// What the model operators' kernels (embedding.hip, qk_rope.hip, distill.hip) share: element types, accesses of 2 to 16
// bytes, reductions over a wave of 64 lanes, and the launch helpers of their host side.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
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

// kN elements that stay packed in their registers (element by element, 16-bit values take a register each).
template <typename T, int kN>
struct Pack {
  using raw_t = typename RawOf<kN * static_cast<int>(sizeof(T))>::type;
  raw_t raw;
  static __device__ __forceinline__ Pack load(const T* at) { return Pack{*reinterpret_cast<const raw_t*>(at)}; }
  __device__ __forceinline__ void store(T* at) const { *reinterpret_cast<raw_t*>(at) = raw; }
  __device__ __forceinline__ void store_nt(T* at) const { __builtin_nontemporal_store(raw, reinterpret_cast<raw_t*>(at)); }

  __device__ __forceinline__ void get(float* f) const {
    if constexpr (kN * sizeof(T) == 2) {
      f[0] = static_cast<float>(__builtin_bit_cast(T, raw));
    } else {
      constexpr int kWords = kN * static_cast<int>(sizeof(T)) / 4;
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        uint32_t word;  // a copy: this compiler casts a vector's first element when given raw[i] itself
        if constexpr (kWords == 1) word = raw;
        else word = raw[i];
        if constexpr (sizeof(T) == 4) {
          f[i] = __uint_as_float(word);
        } else {
          typedef T pair __attribute__((ext_vector_type(2)));
          typedef float pair32 __attribute__((ext_vector_type(2)));
          const pair32 x = __builtin_convertvector(__builtin_bit_cast(pair, word), pair32);
          f[2 * i] = x[0];
          f[2 * i + 1] = x[1];
        }
      }
    }
  }
  __device__ __forceinline__ void set(const float* f) {
    if constexpr (kN * sizeof(T) == 2) {
      raw = __builtin_bit_cast(raw_t, static_cast<T>(f[0]));
    } else {
      constexpr int kWords = kN * static_cast<int>(sizeof(T)) / 4;
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        uint32_t word;
        if constexpr (sizeof(T) == 4) {
          word = __float_as_uint(f[i]);
        } else {
          typedef T pair __attribute__((ext_vector_type(2)));
          typedef float pair32 __attribute__((ext_vector_type(2)));
          word = __builtin_bit_cast(uint32_t, __builtin_convertvector(pair32{f[2 * i], f[2 * i + 1]}, pair));
        }
        if constexpr (kWords == 1) raw = word;
        else raw[i] = word;
      }
    }
  }
};

typedef RawOf<16>::type Vec16;
template <typename T>
constexpr int per_vec() { return 16 / static_cast<int>(sizeof(T)); }
template <typename T>
__device__ __forceinline__ void unpack16(const Vec16& raw, float (&f)[per_vec<T>()]) { Pack<T, per_vec<T>()>{raw}.get(f); }
template <typename T>
__device__ __forceinline__ Vec16 pack16(const float (&f)[per_vec<T>()]) {
  Pack<T, per_vec<T>()> p;
  p.set(f);
  return p.raw;
}

// A stretch of memory for buffer accesses: one register of offsets for many accesses (the rest of an address is scalar), loads
// behind its end give zeros and stores there do nothing. Only the vector operand is promised to be compared with the end, so the
// scalar part of an offset moves the stretch's beginning and shortens it; the instruction's own scalar operand stays zero.
struct Stretch {
  char* base;
  int bytes;
};
__device__ __forceinline__ Stretch stretch(const void* base, int bytes) { return Stretch{static_cast<char*>(const_cast<void*>(base)), bytes}; }
__device__ __forceinline__ __amdgpu_buffer_rsrc_t behind(const Stretch& s, int offset) {
  return __builtin_amdgcn_make_buffer_rsrc(s.base + offset, 0, std::max(s.bytes - offset, 0), 0x00027000);  // raw, 32-bit elements
}
constexpr int kStream = 2;  // the accesses' cache policy: non-temporal
__device__ __forceinline__ Vec16 load16(const Stretch& from, int lane_offset, int offset) {
  return __builtin_amdgcn_raw_buffer_load_b128(behind(from, offset), lane_offset, 0, kStream);
}
__device__ __forceinline__ void store16(const Vec16& v, const Stretch& to, int lane_offset, int offset) {
  __builtin_amdgcn_raw_buffer_store_b128(v, behind(to, offset), lane_offset, 0, kStream);
}

// Reductions over the 64 lanes of a wave by DPP: sums along the rows of 16 lanes, then rows 0 and 2 into 1 and 3, then the lower
// half into the upper; lane 63 has the total, which every lane gets through a scalar register.
template <int kCtrl, int kRows, class F>
__device__ __forceinline__ float dpp_step(float x, float none, F f) {
  return f(x, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(x), kCtrl, kRows, 0xf, false)));
}
struct Add { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct Max { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };
template <class F>
__device__ __forceinline__ float over_16(float x, float none, F f) {  // lane 15 of every row of 16
  x = dpp_step<0x111, 0xf>(x, none, f);
  x = dpp_step<0x112, 0xf>(x, none, f);
  x = dpp_step<0x114, 0xf>(x, none, f);
  return dpp_step<0x118, 0xf>(x, none, f);
}
template <class F>
__device__ __forceinline__ float over_wave(float x, float none, F f) {
  x = over_16(x, none, f);
  x = dpp_step<0x142, 0xa>(x, none, f);
  x = dpp_step<0x143, 0xc>(x, none, f);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
// A value that is the same in all lanes, in a scalar register.
__device__ __forceinline__ float uniform(float x) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x))); }

// Over every row of 16 lanes, every lane gets it: neighbours, pairs, mirrored quads, mirrored eights.
template <class F>
__device__ __forceinline__ float all_16(float x, F f) {
  x = dpp_step<0xb1, 0xf>(x, x, f);
  x = dpp_step<0x4e, 0xf>(x, x, f);
  x = dpp_step<0x141, 0xf>(x, x, f);
  return dpp_step<0x140, 0xf>(x, x, f);
}
__device__ __forceinline__ float wave_sum(float x) { return over_wave(x, 0.0f, Add{}); }
__device__ __forceinline__ float wave_max(float x) { return over_wave(x, -__builtin_inff(), Max{}); }

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
