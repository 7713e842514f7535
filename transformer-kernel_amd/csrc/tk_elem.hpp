// The two 16-bit element types of the serving kernels, and their matrix products.
#pragma once
#include "tk_common.hpp"

namespace tk {

typedef __bf16 bf16;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Workgroups of 256 threads in a launch, which holds fewer than 2^32 threads.
constexpr int64_t kMaxGroups = (1 << 24) - 8;

template <typename T>
struct Elem;

template <>
struct Elem<f16> {
  typedef f16x4 x4;
  typedef f16x8 x8;
  static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma32(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  // c + the sum of a's values, two to an instruction
  static __device__ __forceinline__ float sum8(x8 a, float c) {
    const hf16x2 one = {(__fp16)1.f, (__fp16)1.f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) c = __builtin_amdgcn_fdot2(__builtin_bit_cast(hf16x2, f16x2{a[i], a[i + 1]}), one, c, false);
    return c;
  }
};

template <>
struct Elem<bf16> {
  typedef bf16x4 x4;
  typedef bf16x8 x8;
  static __device__ __forceinline__ f32x4 mfma16(x8 a, x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16 mfma32(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float sum8(x8 a, float c) {
    const bf16x2 one = {(bf16)1.f, (bf16)1.f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) c = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{a[i], a[i + 1]}, one, c, false);
    return c;
  }
};

}  // namespace tk
