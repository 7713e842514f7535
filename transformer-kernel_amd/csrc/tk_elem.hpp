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

// Softmax weights are 2^(x - m), x a score in units of log2 and m a row's reference, the same for O and the sums, so
// that it cancels.  fp16 holds no more than 2^16 and rounds with fewer bits below 2^-14, in steps of 2^-24: with m the
// largest score itself 100000 weights of 2^-25 beside one of 1 would all be 0.  So m lies UP below the largest score:
// weights up to 2^UP.  bf16 has fp32's exponents and needs none of it.  `top` is raw: log2 scores are raw * c, c = s[0].
// For fp16 m is rounded up (s[1] and s[2]: the next numbers above and below c), so that no weight passes 2^UP where
// the scores are so large that half a step of m is one and more.
template <typename T, int UP>
__device__ __forceinline__ float weight_ref(float top, const float (&s)[3]) {
  if constexpr (__is_same(T, f16)) return fmaxf(fmaf(top, s[1], -(float)UP), fmaf(top, s[2], -(float)UP));
  else return top * s[0];
}
constexpr float kMaxScale = 2.3e38f;  // c stays finite: an infinite one would make a score of 0 NaN
inline void set_scales(float (&s)[3], float scale) {
  s[0] = scale * 1.4426950408889634f;
  s[1] = __builtin_nextafterf(s[0], INFINITY);
  s[2] = __builtin_nextafterf(s[0], 0.f);
}

}  // namespace tk
