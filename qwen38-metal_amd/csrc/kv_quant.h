// Quantisers of the KV caches, shared by the kernels that append.
#pragma once
#include <float.h>

#include "common.h"

namespace qm {

// Maximum over the 16 lanes of a DPP row.
__device__ __forceinline__ float row_allmax(float v) {
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, false)));
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, false)));
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xF, 0xF, false)));
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, false)));
}

__device__ __forceinline__ uint32_t pack_q8x4(const int8_t (&qv)[4]) {
  return (uint32_t)(uint8_t)qv[0] | ((uint32_t)(uint8_t)qv[1] << 8) | ((uint32_t)(uint8_t)qv[2] << 16) |
         ((uint32_t)(uint8_t)qv[3] << 24);
}

// Quantises values as qwen38_q8_kv_append does, given the row's absmax:
// s = max(absmax / 127, FLT_MIN), q = round-half-away(clamp(x / s, -127,
// 127)), IEEE division.  Returns s.
__device__ __forceinline__ float q8_quant_with(float amax, const float (&vals)[4], int8_t (&qv)[4]) {
  const float s = fmaxf(amax / 127.0f, FLT_MIN);
#pragma unroll
  for (int i = 0; i < 4; ++i) qv[i] = (int8_t)roundf(fminf(fmaxf(vals[i] / s, -127.0f), 127.0f));
  return s;
}

// One row held 4 values per lane of the wave.
__device__ __forceinline__ float q8_quant_vals(const float (&vals)[4], int8_t (&qv)[4]) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(vals[i]));
  return q8_quant_with(wave_allmax(amax), vals, qv);
}

// Rows held 4 values per lane of G (1, 2 or 4) DPP rows each.
__device__ __forceinline__ float q8_rows_quant(const float (&vals)[4], uint32_t G, int8_t (&qv)[4]) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(vals[i]));
  amax = row_allmax(amax);
  if (G > 1) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(amax), __float_as_uint(amax), false, false);
    amax = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
  }
  if (G > 2) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(amax), __float_as_uint(amax), false, false);
    amax = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
  }
  return q8_quant_with(amax, vals, qv);
}

// A group of the 4-bit cache held 4 values per lane of a DPP row (elements d0 ..
// d0 + 3, those from D on not its own): returns its scale word (s in the low, m in
// the high half), and the codes, -8..7.
__device__ __forceinline__ uint32_t q4kv_group(const float (&x)[4], uint32_t d0, uint32_t D, int (&c)[4]) {
  float top = -INFINITY, low = -INFINITY;  // of x, and of -x
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (d0 + e >= D) continue;
    top = fmaxf(top, x[e]);
    low = fmaxf(low, -x[e]);
    bad |= !(fabsf(x[e]) < INFINITY);
  }
  if (bad) top = INFINITY;  // (a maximum passes NaN over)
  top = row_allmax(top);
  low = row_allmax(low);
  if (!(fabsf(top) < INFINITY)) {  // NaN; and zeros in a group past D
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = 0;
    return top > 0.0f ? 0x7FC07FC0u : 0u;
  }
  // Halves: the difference of any two finite values is finite.
  const uint32_t sb = f32_to_bf16(fmaxf((top * 0.5f + low * 0.5f) / 7.5f, FLT_MIN));
  const float s = bf16_to_f32(sb);
  const uint32_t mb = f32_to_bf16(s * 8.0f - low);
  const float m = bf16_to_f32(mb);
  if (!(fabsf(m) < INFINITY)) {  // (a middle past bf16's range)
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = 0;
    return 0x7FC07FC0u;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float t = (x[e] - m) / s;
    c[e] = d0 + e < D ? (int)rintf(fminf(fmaxf(t, -8.0f), 7.0f)) : 0;
  }
  return sb | mb << 16;
}

// Eight codes of a K word as bf16 of 128 + (c + 8), in order: 0x4300 | u is the bf16
// 128 + u.  Both constants in registers that the compiler cannot see through: it
// then takes one AND-OR a pair (two literals would make it two operations).
struct Q4KvUnpack {
  uint32_t mask = 0x000F000Fu, one = 0x43004300u;
  __device__ __forceinline__ Q4KvUnpack() { asm("" : "+s"(mask), "+v"(one)); }
  __device__ __forceinline__ u32x4 operator()(uint32_t w) const {
    return u32x4{(w & mask) | one, ((w >> 4) & mask) | one, ((w >> 8) & mask) | one, ((w >> 12) & mask) | one};
  }
};

// What a code stands for (the product is exact: one rounding).
__device__ __forceinline__ float q4kv_value(int c, uint32_t word) {
  return __builtin_fmaf((float)c, bf16_to_f32(word & 0xFFFFu), __uint_as_float(word & 0xFFFF0000u));
}

// Sine and cosine in fp64: the angle reduced by quarter turns (pi / 2 in two parts),
// then Taylor series on [-pi/4, pi/4], whose first term left out is below 2e-14.
__device__ __forceinline__ void sincos_f64(double angle, double* sn, double* cs) {
  const double n = rint(angle * 0.6366197723675814);
  double r = fma(-n, 1.5707963267948966, angle);
  r = fma(-n, 6.123233995736766e-17, r);
  const double z = r * r;
  double s = 1.0 / 6227020800.0;
  s = fma(s, z, -1.0 / 39916800.0);
  s = fma(s, z, 1.0 / 362880.0);
  s = fma(s, z, -1.0 / 5040.0);
  s = fma(s, z, 1.0 / 120.0);
  s = fma(s, z, -1.0 / 6.0);
  s = fma(s * z, r, r);
  double c = -1.0 / 87178291200.0;
  c = fma(c, z, 1.0 / 479001600.0);
  c = fma(c, z, -1.0 / 3628800.0);
  c = fma(c, z, 1.0 / 40320.0);
  c = fma(c, z, -1.0 / 720.0);
  c = fma(c, z, 1.0 / 24.0);
  c = fma(c, z, -0.5);
  c = fma(c, z, 1.0);
  const int q = (int)(long long)n & 3;
  *sn = q & 1 ? c : s;
  *cs = q & 1 ? s : c;
  if (q & 2) *sn = -*sn;
  if ((q + 1) & 2) *cs = -*cs;
}

}  // namespace qm
