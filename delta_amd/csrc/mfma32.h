// 32x32 MFMA tiles of the prompt-sized attention kernels (prefill.hip, prefix_attention.hip).
#pragma once

#include "delta_common.h"

namespace delta {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short ps4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) ps4_t lds_ps4_t;

template <int DT>
struct Mfma32;
template <>
struct Mfma32<DELTA_BF16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  __device__ __forceinline__ static f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};
template <>
struct Mfma32<DELTA_FP16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  __device__ __forceinline__ static f32x16 run(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
};

// Two floats -> two packed 16-bit values, round to nearest even (one v_cvt_pk_* on gfx950).
template <int DT>
__device__ __forceinline__ uint32_t pack2(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack2<DELTA_BF16>(float x, float y) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x, y}), b2));
}
template <>
__device__ __forceinline__ uint32_t pack2<DELTA_FP16>(float x, float y) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x, y}), h2));
}

// max / sum of a value and its copy in lane l ^ 32
__device__ __forceinline__ float halves_max(float v) {
  auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(x[0]) + __uint_as_float(x[1]);
}

}  // namespace delta
