// Wave-wide exchanges and reductions without LDS.
#pragma once

#include <hip/hip_runtime.h>
#include <type_traits>

namespace rehip {

// v of lane (lane ^ OFF) without the LDS pipe: v_permlane32_swap / v_permlane16_swap exchange
// 32- / 16-lane halves (each returns both halves; the lane keeps the one that came from its
// partner), DPP row moves do the rest (row_ror:8 = xor 8 within a 16-lane row, quad_perm
// [3,2,1,0] then row_half_mirror = xor 4, quad_perm [2,3,0,1] / [1,0,3,2] = xor 2 / xor 1).
// The pairs are those of __shfl_xor(v, OFF, 64), so a butterfly over them keeps its bits.
template <int OFF>
__device__ __forceinline__ float lane_xor(float v) {
  const int u = __float_as_int(v);
  if constexpr (OFF == 32) {
    const auto s = __builtin_amdgcn_permlane32_swap((unsigned)u, (unsigned)u, false, false);
    return __uint_as_float((threadIdx.x & 32) ? s[0] : s[1]);
  } else if constexpr (OFF == 16) {
    const auto s = __builtin_amdgcn_permlane16_swap((unsigned)u, (unsigned)u, false, false);
    return __uint_as_float((threadIdx.x & 16) ? s[0] : s[1]);
  } else if constexpr (OFF == 8) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, u, 0x128, 0xF, 0xF, false));
  } else if constexpr (OFF == 4) {
    const int r = __builtin_amdgcn_update_dpp(0, u, 0x1B, 0xF, 0xF, false);
    return __int_as_float(__builtin_amdgcn_update_dpp(0, r, 0x141, 0xF, 0xF, false));
  } else if constexpr (OFF == 2) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, u, 0x4E, 0xF, 0xF, false));
  } else {
    static_assert(OFF == 1, "lane_xor: OFF is a power of two up to 32");
    return __int_as_float(__builtin_amdgcn_update_dpp(0, u, 0xB1, 0xF, 0xF, false));
  }
}
template <int OFF>
__device__ __forceinline__ unsigned lane_xor_u32(unsigned v) {
  return __float_as_uint(lane_xor<OFF>(__uint_as_float(v)));
}
// f(OFF) for the butterfly's pairs: lanes xor 32, 16, .., 1
template <class F>
__device__ __forceinline__ void wave_butterfly(F f) {
  f(std::integral_constant<int, 32>{});
  f(std::integral_constant<int, 16>{});
  f(std::integral_constant<int, 8>{});
  f(std::integral_constant<int, 4>{});
  f(std::integral_constant<int, 2>{});
  f(std::integral_constant<int, 1>{});
}
// butterfly max / sum over the wave (every lane ends with the result), pairs xor 32, 16, .., 1
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, lane_xor<32>(v));
  v = fmaxf(v, lane_xor<16>(v));
  v = fmaxf(v, lane_xor<8>(v));
  v = fmaxf(v, lane_xor<4>(v));
  v = fmaxf(v, lane_xor<2>(v));
  return fmaxf(v, lane_xor<1>(v));
}
__device__ __forceinline__ float wave_sum(float v) {
  v += lane_xor<32>(v);
  v += lane_xor<16>(v);
  v += lane_xor<8>(v);
  v += lane_xor<4>(v);
  v += lane_xor<2>(v);
  return v + lane_xor<1>(v);
}

// inclusive sums over the lanes of a wave
__device__ __forceinline__ int wave_scan(int v) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(v, off, 64);
    if ((int)(threadIdx.x & 63) >= off) v += y;
  }
  return v;
}

// The sum over a workgroup of WAVES waves, and in `before` that of the threads below this one.
template <int WAVES>
__device__ __forceinline__ int scan_block(int v, int& before) {
  __shared__ int part[WAVES];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, inc = wave_scan(v);
  if (lane == 63) part[w] = inc;
  __syncthreads();
  int all = 0;
  before = inc - v;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    before += i < w ? part[i] : 0;
    all += part[i];
  }
  __syncthreads();
  return all;
}

// What the wave's lanes wrote to LDS before this, all its lanes read after it. LDS serves a wave in order, so this is
// no instruction: it keeps the compiler from moving or reusing reads across it.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

}  // namespace rehip
