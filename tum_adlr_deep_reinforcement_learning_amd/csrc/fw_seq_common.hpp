// fw_seq_common.hpp -- element types, wide loads and small helpers of the sequence kernels (fw_sequence.hip,
// fw_groupnorm.hip).
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "../../include/fwrollout.h"
#include "../../include/fwsim.h"

namespace fw {
int set_error(int code, const std::string& msg);
}

#define FW_HIP(expr)                                                                                     \
  do {                                                                                                   \
    hipError_t e_ = (expr);                                                                              \
    if (e_ != hipSuccess) return fw::set_error(FW_E_HIP, std::string(#expr ": ") + hipGetErrorString(e_)); \
  } while (0)

namespace fwseq {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct bf16 {  // storage only; arithmetic is in float
  uint16_t u;
};
struct f16 {
  _Float16 h;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __uint_as_float((uint32_t)x.u << 16); }
__device__ __forceinline__ float to_f32(f16 x) { return (float)x.h; }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float x) {  // to nearest, ties to even (the hardware's conversion)
  return bf16{__builtin_bit_cast(uint16_t, (__bf16)x)};
}
template <>
__device__ __forceinline__ f16 from_f32<f16>(float x) {
  return f16{(_Float16)x};
}

// two floats as a pair of bfloat16 (to nearest), and the halves of a pair as floats
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
}
__device__ __forceinline__ float lo_f32(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float hi_f32(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// n elements moved as one access of up to 16 bytes
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T e[N];
};

template <typename T>
constexpr int vec_elems(int n) {  // elements of one access when n contiguous ones are wanted
  return n * (int)sizeof(T) <= 16 ? n : 16 / (int)sizeof(T);
}

template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float* out) {
  const Pack<T, N> v = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; i++) out[i] = to_f32(v.e[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float* x) {
  Pack<T, N> v;
#pragma unroll
  for (int i = 0; i < N; i++) v.e[i] = from_f32<T>(x[i]);
  *reinterpret_cast<Pack<T, N>*>(p) = v;
}

}  // namespace fwseq
