// Microscaled rows (OCP MX): blocks of 32 consecutive values share a power-of-two scale.
//
//   top   = max |v| of the block
//   byte  = max(floor(log2 top) - emax + 127, 0)       emax: 8 for e4m3, 2 for e2m1
//   code  = v / 2^(byte - 127) to nearest, ties to even, saturated at 448 (e4m3) or 6 (e2m1)
//
// A block that holds an infinity or a NaN has the byte 255, which stands for NaN: all its
// values read back, and every product with it, as NaN. Rows are stored padded with zeros to a
// multiple of 128 values, so that a product's loop over a row has no tail.
#pragma once

#include "fm_device.h"

namespace fm {

constexpr int MX_BLOCK = 32;
constexpr int MX_PAD = 128;

__host__ __device__ __forceinline__ int64_t mx_padded(int64_t cols) { return (cols + MX_PAD - 1) / MX_PAD * MX_PAD; }

// The magnitude bits of a float: as integers they order finite values, infinity and NaN, so
// that an integer maximum loses none of them.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The scale byte of a block whose largest magnitude has the bits `top` (a subnormal has the
// exponent field 0 and ends at byte 0, as every top below 2^(emax - 126) does).
template <int BITS>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
  const int e = (int)(top >> 23);
  if (e == 255) return 255u;
  const int b = e - (BITS == 8 ? 8 : 2);
  return b > 0 ? (uint32_t)b : 0u;
}
// 2^(byte - 127) as a float (2^-127 is subnormal; 255 gives 1, its block's codes do not count).
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x3f800000u : byte == 0u ? 0x00400000u : byte << 23);
}

// v_cvt_scalef32_* divide by the scale and round to nearest even; e2m1 saturates by itself,
// e4m3 would give NaN past 464.
__device__ __forceinline__ uint32_t mx_pack_e4m3x4(float v0, float v1, float v2, float v3, float scale) {
  typedef __attribute__((ext_vector_type(2))) short s16x2_t;
  const float lim = 448.f * scale;
  auto sat = [&](float v) { return __builtin_amdgcn_fmed3f(v, -lim, lim); };
  s16x2_t w = {0, 0};
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, sat(v0), sat(v1), scale, false);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, sat(v2), sat(v3), scale, true);
  return __builtin_bit_cast(uint32_t, w);
}
__device__ __forceinline__ uint32_t mx_pack_e2m1x8(const float (&v)[8], float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
}

}  // namespace fm
