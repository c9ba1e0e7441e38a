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

// The same of four values at once; all 64 lanes take part.  (A DPP operand is read two
// wait states after its register was written at the earliest.)
__device__ __forceinline__ void row_allmax4(float (&v)[4]) {
#define QM_STEP(how) QM_MAX(0, how) QM_MAX(1, how) QM_MAX(2, how) QM_MAX(3, how)
#define QM_MAX(r, how) "v_max_f32_dpp %" #r ", %" #r ", %" #r " " how " row_mask:0xf bank_mask:0xf\n"
  asm("s_nop 1\n" QM_STEP("quad_perm:[1,0,3,2]") QM_STEP("quad_perm:[2,3,0,1]") QM_STEP("row_ror:4") QM_STEP("row_ror:8")
      : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
#undef QM_MAX
#undef QM_STEP
}

// The groups of a key (x[0]) and of a value (x[1]) in the 4-bit cache, held 4 elements
// per lane of a DPP row: d0 .. d0 + 3, those from D on not the group's own (WHOLE: all
// or none are).  Gives the scale words (s in the low, m in the high half) and the
// codes + 8.  All 64 lanes take part.
//
// Quotients round as divisions do: by a reciprocal and one step on the remainder, both
// exact but for their last rounding.
template <bool WHOLE>
__device__ __forceinline__ void q4kv_groups(const float (&x)[2][4], uint32_t d0, uint32_t D, uint32_t (&word)[2],
                                            uint32_t (&u)[2][4]) {
  float stat[4];  // maxima of x[0], -x[0], x[1], -x[1]
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float top, low, z = x[k][0] * 0.0f;
    if constexpr (WHOLE) {
      asm("v_max_f32 %0, %4, %5\nv_max_f32 %1, -%4, -%5\nv_max3_f32 %0, %2, %3, %0\nv_max3_f32 %1, -%2, -%3, %1"
          : "=&v"(top), "=&v"(low)
          : "v"(x[k][0]), "v"(x[k][1]), "v"(x[k][2]), "v"(x[k][3]));
      if (d0 >= D) top = low = -INFINITY;
    } else {
      top = low = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        top = fmaxf(top, d0 + e < D ? x[k][e] : -INFINITY);
        low = fmaxf(low, d0 + e < D ? -x[k][e] : -INFINITY);
      }
    }
#pragma unroll
    for (int e = 1; e < 4; ++e) z = __builtin_fmaf(x[k][e], 0.0f, z);
    stat[2 * k] = z == 0.0f ? top : INFINITY;  // (a maximum passes NaN over)
    stat[2 * k + 1] = low;
  }
  row_allmax4(stat);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float top = stat[2 * k], low = stat[2 * k + 1];
    // Halves: the difference of any two finite values is finite.  Small ones are scaled
    // up, so that no remainder is lost.
    const float h0 = top * 0.5f + low * 0.5f;
    const bool tiny = h0 < 0x1p-60f;
    const float h = tiny ? h0 * 0x1p64f : h0, r75 = 1.0f / 7.5f;
    float q = h * r75;
    q = __builtin_fmaf(__builtin_fmaf(-q, 7.5f, h), r75, q);
    const uint32_t sb = f32_to_bf16(fmaxf(tiny ? q * 0x1p-64f : q, FLT_MIN));
    const uint32_t mb = f32_to_bf16(__builtin_fmaf(bf16_to_f32(sb), 8.0f, -low));
    const float m = bf16_to_f32(mb);
    // Not fine: a value that is not finite, a middle past bf16's range, or no element.
    const bool fine = fabsf(top) < INFINITY && fabsf(m) < INFINITY;
    word[k] = fine ? sb | mb << 16 : top == -INFINITY ? 0u : 0x7FC07FC0u;
    // (x - m) / s with s = sn 2^e, sn in [1, 2) (of 8 bits: no reciprocal lies near a
    // border); its codes by the rounding of a sum with 1.5 2^23.
    const int e2 = 127 - (int)(sb >> 7);
    const float sn = __uint_as_float((sb & 0x7Fu) << 16 | 0x3F800000u);
    float r = __builtin_amdgcn_rcpf(sn);
    r = __builtin_fmaf(__builtin_fmaf(-sn, r, 1.0f), r, r);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = __builtin_amdgcn_ldexpf(x[k][e] - m, e2), t0 = a * r;
      const float t = __builtin_fmaf(__builtin_fmaf(-t0, sn, a), r, t0);
      const uint32_t c = __float_as_uint(__builtin_amdgcn_fmed3f(t, -8.0f, 7.0f) + 12582920.0f) & 15;
      u[k][e] = fine && d0 + (WHOLE ? 0 : e) < D ? c : 8u;
    }
  }
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
