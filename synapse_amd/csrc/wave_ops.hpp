// Reductions over a wave by lane moves (no trip through LDS).
#pragma once

#include "common.hpp"

namespace syn {

// x of a partner lane: steps 1 to 32 together reach every lane of the wave, by
// lane moves (no trip through LDS); what steps O, O / 2, ... have combined is
// the same in all lanes that they connect
template <int STEP> __device__ __forceinline__ uint32_t partner(uint32_t x) {
  if constexpr (STEP == 32 || STEP == 16) {
    const auto p = STEP == 32 ? __builtin_amdgcn_permlane32_swap(x, x, false, false)
                              : __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return threadIdx.x & STEP ? p[0] : p[1];
  } else {
    // row_mirror, row_half_mirror, two quad permutations
    constexpr int ctl = STEP == 8 ? 0x140 : (STEP == 4 ? 0x141 : (STEP == 2 ? 0x4e : 0xb1));
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctl, 0xf, 0xf, false);
  }
}
template <int STEP> __device__ __forceinline__ int partner(int x) { return (int)partner<STEP>((uint32_t)x); }
template <int STEP> __device__ __forceinline__ float partner(float x) {
  return __uint_as_float(partner<STEP>(__float_as_uint(x)));
}
template <int STEP> __device__ __forceinline__ double partner(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  const uint64_t lo = partner<STEP>((uint32_t)u), hi = partner<STEP>((uint32_t)(u >> 32));
  return __longlong_as_double((long long)(hi << 32 | lo));
}
template <class F, class Op> __device__ __forceinline__ F over_wave(F x, Op op) {
  x = op(x, partner<32>(x));
  x = op(x, partner<16>(x));
  x = op(x, partner<8>(x));
  x = op(x, partner<4>(x));
  x = op(x, partner<2>(x));
  return op(x, partner<1>(x));
}
__device__ __forceinline__ float greater(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double greater(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ float lesser(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double lesser(double a, double b) { return fmin(a, b); }
template <class F> __device__ __forceinline__ F wave_max(F x) {
  return over_wave(x, [](F a, F b) { return greater(a, b); });
}
template <class F> __device__ __forceinline__ F wave_sum(F x) {
  return over_wave(x, [](F a, F b) { return a + b; });
}

// x of the lane that a DPP control names, 0 where there is none
template <int CTL, int ROWS> __device__ __forceinline__ uint32_t from_lane(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTL, ROWS, 0xf, false);
}
template <int CTL, int ROWS> __device__ __forceinline__ int from_lane(int x) {
  return (int)from_lane<CTL, ROWS>((uint32_t)x);
}
template <int CTL, int ROWS> __device__ __forceinline__ double from_lane(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  const uint64_t lo = from_lane<CTL, ROWS>((uint32_t)u), hi = from_lane<CTL, ROWS>((uint32_t)(u >> 32));
  return __longlong_as_double((long long)(hi << 32 | lo));
}
// the sum over the lanes up to this one: within the rows of 16 by shifts of 1, 2, 4
// and 8, then row 0's to row 1 and 2's to 3, then that of both to the upper two
template <class F> __device__ __forceinline__ F wave_upto(F x) {
  x += from_lane<0x111, 0xf>(x);
  x += from_lane<0x112, 0xf>(x);
  x += from_lane<0x114, 0xf>(x);
  x += from_lane<0x118, 0xf>(x);
  x += from_lane<0x142, 0xa>(x);
  return x + from_lane<0x143, 0xc>(x);
}
// the sum over the lanes below this one, given that up to it
template <class F> __device__ __forceinline__ F wave_shifted(F upto) { return from_lane<0x138, 0xf>(upto); }

}  // namespace syn
