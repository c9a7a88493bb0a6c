// qr_lanes.h -- exchanges between the lanes of a wave without LDS.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qr {

// The value of the lane whose number differs by the bits of X: 1, 2, 3 within a
// quad, 7 and 15 mirrored halves of a row and rows, 8 a row turned by half, 16
// and 32 by swapping rows.  All lanes active.
template <int X>
__device__ inline uint32_t lane_xor(uint32_t v) {
  constexpr int kCtrl = X == 1 ? 0xB1 : X == 2 ? 0x4E : X == 3 ? 0x1B : X == 7 ? 0x141
                      : X == 15 ? 0x140 : 0x128;
  if constexpr (X == 4) {
    return lane_xor<3>(lane_xor<7>(v));
  } else if constexpr (X == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  } else if constexpr (X == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? r[0] : r[1];
  } else if constexpr (X == 31) {
    return lane_xor<15>(lane_xor<16>(v));
  } else if constexpr (X == 63) {
    return lane_xor<31>(lane_xor<32>(v));
  } else {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xF, 0xF, true);
  }
}
template <int X>
__device__ inline float lane_xor_f(float v) {
  return __builtin_bit_cast(float, lane_xor<X>(__builtin_bit_cast(uint32_t, v)));
}
template <int X>
__device__ inline unsigned long long lane_xor_64(unsigned long long k) {
  return (unsigned long long)lane_xor<X>((uint32_t)(k >> 32)) << 32 | lane_xor<X>((uint32_t)k);
}

// Both values of each pair of lanes that differ by 16 (by 32), in all lanes.  (They are
// copied out of the builtin's vector before they are reinterpreted: a bit cast of an element
// itself takes element 0.)
__device__ inline void pair16(float v, float* x, float* y) {
  const uint32_t a = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const uint32_t p = r[0], q = r[1];
  *x = __builtin_bit_cast(float, p);
  *y = __builtin_bit_cast(float, q);
}
__device__ inline void pair32(float v, float* x, float* y) {
  const uint32_t a = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  const uint32_t p = r[0], q = r[1];
  *x = __builtin_bit_cast(float, p);
  *y = __builtin_bit_cast(float, q);
}
// The larger of two numbers, NaN where one is: one instruction, where fmaxf of values that came
// by way of memory or another lane takes three.
__device__ inline float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Over the four lanes of equal lane % 16.
__device__ inline float rows_max(float v) {
  float x, y;
  pair16(v, &x, &y);
  pair32(fmaxf(x, y), &x, &y);
  return fmaxf(x, y);
}
__device__ inline float rows_larger(float v) {
  float x, y;
  pair16(v, &x, &y);
  pair32(larger(x, y), &x, &y);
  return larger(x, y);
}
__device__ inline float rows_sum(float v) {
  float x, y;
  pair16(v, &x, &y);
  pair32(x + y, &x, &y);
  return x + y;
}

// Over the 16 lanes of a row.
__device__ inline float row_max(float v) {
  v = fmaxf(v, lane_xor_f<1>(v));
  v = fmaxf(v, lane_xor_f<2>(v));
  v = fmaxf(v, lane_xor_f<7>(v));
  return fmaxf(v, lane_xor_f<15>(v));
}
__device__ inline float row_sum(float v) {
  v += lane_xor_f<1>(v);
  v += lane_xor_f<2>(v);
  v += lane_xor_f<7>(v);
  return v + lane_xor_f<15>(v);
}
// Over the wave.
__device__ inline float wave_max(float v) { return rows_max(row_max(v)); }
__device__ inline float wave_sum(float v) { return rows_sum(row_sum(v)); }

}  // namespace qr
