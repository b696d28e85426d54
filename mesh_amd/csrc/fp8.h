// Shared by the sources of the 8-bit operands (gfx950 only).
#pragma once

#include "../../include/mesh_moe_fp8.h"
#include "common.h"

namespace mesh_moe {

constexpr int FP8_BLOCK = 128;    // values that share a scale
constexpr int FP8_UNIT = 127;     // the scale byte of 2^0
constexpr int64_t MAX_THREADS = 0xffffffffLL;   // of a launch, in one dimension

// bytes of a row of K values, and of its scales
__host__ __device__ __forceinline__ int64_t fp8_row_bytes(int K) {
  return ((int64_t)K + FP8_BLOCK - 1) / FP8_BLOCK * FP8_BLOCK;
}
__host__ __device__ __forceinline__ int64_t fp8_scale_bytes(int K) {
  return (((int64_t)K + FP8_BLOCK - 1) / FP8_BLOCK + 3) / 4 * 4;
}

// A block's scale from `top`, the bits of its largest magnitude (sign removed; the bits
// of magnitudes are ordered as they are).  With top = 1.m * 2^p the exponent is p - 8
// for m <= 3/4 (448 = 1.75 * 2^8) and p - 7 above; adding 0x1fffff carries into the
// exponent's bits for exactly those m.
struct Fp8Scale {
  uint32_t byte;
  float factor;                   // 2^-exponent; NaN for a block that is not finite
};
__device__ __forceinline__ Fp8Scale fp8_scale(uint32_t top) {
  const int at = (int)((top + 0x1fffffu) >> 23) - 8;
  const uint32_t byte = at < 10 ? 10u : (uint32_t)at;       // 2^-117 at least
  Fp8Scale s;
  const bool finite = top < 0x7f800000u;
  s.byte = finite ? byte : (uint32_t)FP8_UNIT;
  s.factor = __uint_as_float(finite ? (254u - byte) << 23 : 0x7fc00000u);
  return s;
}

// four values, already divided by their scale (so at most 448, or NaN), rounded to
// e4m3, ties to even
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
}

__device__ __forceinline__ uint32_t magnitude_bits(float v) {
  return __float_as_uint(v) & 0x7fffffffu;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, true);
}
// The largest of 16 neighbouring lanes, in all of them: pairs, quads, halves, rows.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
  v = max(v, dpp<0xb1>(v));       // quad_perm [1,0,3,2]
  v = max(v, dpp<0x4e>(v));       // quad_perm [2,3,0,1]
  v = max(v, dpp<0x141>(v));      // row_half_mirror
  return max(v, dpp<0x140>(v));   // row_mirror
}

// fp8.hip, for the gradients, which make operands of dy (arguments checked by them).
// only_counted: rows from an expert's count on are left out, but for the columns' first
// two blocks.
int fp8_quantize(const void* x, const void* relu_mask, const int32_t* row_count,
                 void* row_values, uint8_t* row_scales, void* column_values,
                 uint8_t* column_scales, int E, int R, int K, int dtype,
                 bool only_counted, hipStream_t st);

}  // namespace mesh_moe
