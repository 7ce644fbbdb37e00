// Page tables, integers of either width and 16-bit floats, for the kernels on paged caches.
#pragma once

#include "mg_common.h"

namespace {

typedef uint16_t u16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

struct Bf16 {
  u16 x;
};
struct Fp16 {
  _Float16 x;
};
__device__ __forceinline__ float pg_float(Bf16 v) { return __uint_as_float((unsigned)v.x << 16); }
__device__ __forceinline__ float pg_float(Fp16 v) { return (float)v.x; }
__device__ __forceinline__ float pg_float(float v) { return v; }
template <typename T>
__device__ __forceinline__ T pg_round(float v);
template <>
__device__ __forceinline__ Bf16 pg_round<Bf16>(float v) {
  return Bf16{__builtin_bit_cast(u16, (__bf16)v)};
}
template <>
__device__ __forceinline__ Fp16 pg_round<Fp16>(float v) {
  return Fp16{(_Float16)v};
}
template <>
__device__ __forceinline__ float pg_round<float>(float v) {
  return v;
}

// Two values as a word of two elements.
template <typename T>
__device__ __forceinline__ unsigned pg_pack(float x, float y);
template <>
__device__ __forceinline__ unsigned pg_pack<Bf16>(float x, float y) {
  const bf16x2 h = {(__bf16)x, (__bf16)y};
  unsigned u = __builtin_bit_cast(unsigned, h);
  asm("" : "+v"(u));  // keeps the pair one packed conversion
  return u;
}
template <>
__device__ __forceinline__ unsigned pg_pack<Fp16>(float x, float y) {
  const f16x2 h = {(_Float16)x, (_Float16)y};
  return __builtin_bit_cast(unsigned, h);
}

// Integers of a caller: int32, or int64 where wide.
struct Ints {
  const void* p;
  int wide;
  __device__ __forceinline__ int64_t operator[](int64_t i) const {
    return wide ? ((const int64_t*)p)[i] : (int64_t)((const int*)p)[i];
  }
};

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31, as (n m) >> s with s = 31 + ceil(log2 d) and
// m = floor(2^s / d) + 1: m d exceeds 2^s by at most d <= 2^(s - 31), so the product's error
// n (m d - 2^s) / (d 2^s) is below 1 / d, too little to reach the next whole number.
struct Divisor {
  unsigned d, m;
  int s;
};
inline Divisor pg_divisor(int64_t d) {
  int c = 0;
  while ((1ll << c) < d) ++c;
  return Divisor{(unsigned)d, (unsigned)((1ull << (31 + c)) / (unsigned long long)d + 1), 31 + c};
}
__device__ __forceinline__ unsigned pg_div(unsigned n, const Divisor& v) {
  return (unsigned)(((unsigned long long)n * v.m) >> v.s);
}

}  // namespace
