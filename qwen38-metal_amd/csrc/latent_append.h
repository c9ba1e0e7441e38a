// Writing a row of the 8-bit latent cache, for the kernels that append.
//
// A token's row is its latent (rank_pad codes) and the shared key (64 codes),
// each with one fp32 scale: s = max(absmax / 127, FLT_MIN), code = round half
// away(clamp(x / s, -127, 127)) with IEEE division, the quantiser of the Q8 KV
// cache (but that a part with a NaN or an infinity stands for NaN).  The latent
// may be RMS-normalised on its way (x rsqrt(mean x^2 + eps) w), in fp32: the
// projection's row is read once and nothing else is written but the 8 bits.
//
// A wave takes a row: 8 elements per lane of the latent (16 bytes in, 8 out)
// and 8 per lane of lanes 0..7 of the key.
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

// Quantises a wave's row held 8 elements per lane; returns the scale: NaN, with
// codes of 0, for a row that holds a NaN or an infinity.
__device__ __forceinline__ float latent_quantise(const float (&x)[8], u32x2* codes) {
  float amax = 0.0f;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    amax = fmaxf(amax, fabsf(x[i]));
    finite = finite && fabsf(x[i]) <= FLT_MAX;
  }
  if (__any(!finite)) {
    *codes = u32x2{0, 0};
    return __uint_as_float(0x7FC00000u);
  }
  amax = wave_allmax(amax);
  const float s = fmaxf(amax / 127.0f, FLT_MIN);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int8_t c = (int8_t)roundf(fminf(fmaxf(x[i] / s, -127.0f), 127.0f));
    w[i / 4] |= (uint32_t)(uint8_t)c << (8 * (i % 4));
  }
  *codes = u32x2{w[0], w[1]};
  return s;
}

// Row `item` of n becomes token `token` of `to`.
__device__ __forceinline__ void latent_append_row(const LatentNewRows& n, const LatentRows& to, size_t token,
                                                  uint32_t item, uint32_t lane) {
  const uint16_t* src = n.kv + (size_t)item * (n.rank + n.rope);
  const uint32_t e = 8 * lane;
  const u32x4 none = {0, 0, 0, 0};
  const u32x4 lat = e < n.rank ? *(const u32x4*)(src + e) : none;
  const u32x4 key = e < n.rope ? *(const u32x4*)(src + n.rank + e) : none;
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = n.norm && e < n.rank ? n.norm[e + i] : 1.0f;
  float x[8], k[8];
  latent_unpack8(lat, x);
  latent_unpack8(key, k);
  if (n.norm) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
    const float r = 1.0f / sqrtf(wave_allsum(ss) / (float)n.rank + n.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
  }
  u32x2 cx, ck;
  const float sx = latent_quantise(x, &cx), sk = latent_quantise(k, &ck);
  int8_t* row = to.codes + token * (n.rank_pad + kLatentRope);
  if (e < n.rank_pad) *(u32x2*)(row + e) = cx;
  if (e < kLatentRope) *(u32x2*)(row + n.rank_pad + e) = ck;
  if (lane == 0) *(float2*)(to.scales + 2 * token) = float2{sx, sk};
}

}  // namespace qm
