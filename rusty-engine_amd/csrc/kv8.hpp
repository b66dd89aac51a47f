// What the kernels over int8 pages share: codes and f32 operands as f16 operands of the matrix instructions.
#pragma once

#include <hip/hip_runtime.h>

#include "wave.hpp"

namespace rehip {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// eight codes as f16: 0x6400 + u is the f16 value 1024 + u for a byte u = c + 128, less 1152 is c
__device__ __forceinline__ h8 codes8(unsigned a, unsigned b) {
  union { unsigned u[4]; h2 h[4]; h8 v; } r;
  a ^= 0x80808080u;
  b ^= 0x80808080u;
  r.u[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
  r.u[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
  r.u[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
  r.u[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
  const h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
#pragma unroll
  for (int i = 0; i < 4; ++i) r.h[i] += off;
  return r.v;
}

// x = hi + lo, each rounded to the nearest f16. minus_one: -1, but unknown to the compiler, which then subtracts hi in
// one mixed-precision fma instead of converting it back first
__device__ __forceinline__ void split8(const float (&x)[8], float minus_one, h8& hi, h8& lo) {
  union { h2 h[4]; h8 v; } a, b;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a.h[i] = __builtin_convertvector((f32x2{x[2 * i], x[2 * i + 1]}), h2);
    const f32x2 r = {__builtin_fmaf((float)a.h[i][0], minus_one, x[2 * i]),
                     __builtin_fmaf((float)a.h[i][1], minus_one, x[2 * i + 1])};
    b.h[i] = __builtin_convertvector(r, h2);
  }
  hi = a.v;
  lo = b.v;
}

// 2^x for x <= 16: what is below the smallest normal float may come out as 0
__device__ __forceinline__ float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// the largest over the four lanes that share a column of the 16 x 16 layouts (one of the swapped values is the lane's
// own, so both may be taken), and the sum
__device__ __forceinline__ float column_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_sum(float v) {
  v += lane_xor<16>(v);
  return v + lane_xor<32>(v);
}

}  // namespace rehip
