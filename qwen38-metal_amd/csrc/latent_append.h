// Writing a row of the 8-bit latent cache, for the kernels that append.
//
// A token's row is its latent (rank_pad codes) and the shared key (64 codes),
// each with one fp32 scale: s = max(absmax / 127, FLT_MIN), code = round half
// away(clamp(x / s, -127, 127)) with IEEE division, the quantiser of the Q8 KV
// cache (but that a part with a NaN or an infinity stands for NaN).  The latent
// may be RMS-normalised on its way (x rsqrt(mean x^2 + eps) w), in fp32: the
// projection's row is read once and nothing else is written but the 8 bits.
//
// A wave takes R rows: of each latent 8 elements per lane (16 bytes in, 8 out), and
// the R shared keys at once, 8 lanes each.  Sixteen divisions a lane and row would
// bound it, not the memory, so codes come from x times 1 / s wherever that cannot
// differ from the division's: only a quotient within 10^-4 of a half could round
// otherwise (the product is off by 3 * 2^-24 of at most 127), and is divided.  8192
// rows of 512 + 64 with norm, 9.4 MB in and 4.8 out: 10.2 us (one row a wave 12.8;
// dividing always, with a key to a wave, 14.2).
#pragma once
#include <float.h>

#include "common.h"
#include "latent.h"

namespace qm {

__device__ __forceinline__ void latent_unpack8(u32x4 v, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_to_f32(v[i] & 0xFFFFu);
    x[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
  }
}

// The eight elements' magnitudes, the largest, as bits: from 0x7F800000 on there is
// an infinity or a NaN among them.
__device__ __forceinline__ uint32_t latent_top(const float (&x)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  return top;
}
// Codes of eight elements of magnitudes up to 127 s (and what its rounding adds).
__device__ __forceinline__ u32x2 latent_codes(const float (&x)[8], float s) {
  const float inv = 1.0f / s;
  uint32_t c[8];
  float off = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = x[i] * inv, t = v + 12582912.0f;  // 1.5 2^23: the nearest whole number in the low bits
    off = fmaxf(off, fabsf(v - (t - 12582912.0f)));
    c[i] = __float_as_uint(t);
  }
  if (__any(off > 0.4999f)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = (uint32_t)(int)roundf(fminf(fmaxf(x[i] / s, -127.0f), 127.0f));
  }
  u32x2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = perm_b32(perm_b32(c[4 * i + 3], c[4 * i + 2], 0x0C0C0400u), perm_b32(c[4 * i + 1], c[4 * i], 0x0C0C0400u), 0x05040100u);
  return w;
}

// Rows item .. item + R - 1 of n, those below `end`, become tokens from `token` on.
template <int R>
__device__ __forceinline__ void latent_append_rows(const LatentNewRows& n, const LatentRows& to, size_t token,
                                                   uint32_t item, uint32_t end, uint32_t lane) {
  const uint32_t e = 8 * lane, width = n.rank + n.rope, key_row = lane / 8, ke = 8 * (lane % 8);
  const uint16_t* src = n.kv + (size_t)item * width;
  const u32x4 none = {0, 0, 0, 0};
  u32x4 lat[R];
#pragma unroll
  for (int i = 0; i < R; ++i) lat[i] = e < n.rank && item + i < end ? *(const u32x4*)(src + (size_t)i * width + e) : none;
  const bool has_key = key_row < R && item + key_row < end;
  const u32x4 key = has_key && ke < n.rope ? *(const u32x4*)(src + (size_t)key_row * width + n.rank + ke) : none;
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = n.norm && e < n.rank ? n.norm[e + i] : 1.0f;
  const size_t stride = n.rank_pad + kLatentRope;
  int8_t* const rows = to.codes + token * stride;
  float* const scales = to.scales + 2 * token;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (item + i >= end) break;  // wave-uniform
    float x[8];
    latent_unpack8(lat[i], x);
    if (n.norm) {
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
      const float r = 1.0f / sqrtf(wave_allsum(ss) / (float)n.rank + n.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] * r * w[j];
    }
    const uint32_t top = latent_top(x);
    u32x2 codes = none.xy;
    float s = __uint_as_float(0x7FC00000u);  // a row that stands for NaN
    if (!__any(top >= 0x7F800000u)) {
      s = fmaxf(wave_allmax(__uint_as_float(top)) / 127.0f, FLT_MIN);
      codes = latent_codes(x, s);
    }
    if (e < n.rank_pad) *(u32x2*)(rows + i * stride + e) = codes;
    if (lane == 0) scales[2 * i] = s;
  }
  float k[8];
  latent_unpack8(key, k);
  uint32_t top = latent_top(k);
#pragma unroll
  for (int d = 1; d < 8; d *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, d));
  const bool number = top < 0x7F800000u;
#pragma unroll
  for (int i = 0; i < 8; ++i) k[i] = number ? k[i] : 0.0f;
  const float s = fmaxf((number ? __uint_as_float(top) : 0.0f) / 127.0f, FLT_MIN);
  const u32x2 codes = latent_codes(k, s);
  if (!has_key) return;
  *(u32x2*)(rows + key_row * stride + n.rank_pad + ke) = codes;
  if (ke == 0) scales[2 * key_row + 1] = number ? s : __uint_as_float(0x7FC00000u);
}

}  // namespace qm
