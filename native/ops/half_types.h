// The two 16-bit float types of the packed-batch kernels, as tags: storage is
// an unsigned short, arithmetic is fp32, every store rounds to nearest even.
#pragma once
#include "common.h"

namespace kgwe {

struct Bf16 {
  static __device__ __forceinline__ float up(unsigned short v) { return bf2f(v); }
  static __device__ __forceinline__ unsigned short down(float f) { return f2bf(f); }
};

struct Fp16 {
  static __device__ __forceinline__ float up(unsigned short v) {
    return static_cast<float>(__builtin_bit_cast(_Float16, v));
  }
  static __device__ __forceinline__ unsigned short down(float f) {
    return __builtin_bit_cast(unsigned short, static_cast<_Float16>(f));
  }
};

// Type codes of the C entries' `dtype` argument.
constexpr int kTypeBf16 = 0, kTypeFp16 = 1;

}  // namespace kgwe
