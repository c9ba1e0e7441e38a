// Device side of rotary positions, shared by the stand-alone kernel (rotary.hip)
// and the appends that rotate on the way (kv_append.hip).
#pragma once
#include "common.h"
#include "rotary.h"

namespace qm {

__device__ __forceinline__ void unpack8(u32x4 v, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_to_f32(v[i] & 0xFFFFu);
    x[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  u32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = f32_to_bf16(x[2 * i]) | ((uint32_t)f32_to_bf16(x[2 * i + 1]) << 16);
  return v;
}

// Sines and cosines of one position, times `factor`, by `threads` threads: the angle
// in fp64, reduced modulo 2 pi there.
__device__ __forceinline__ void rotary_table(const double* freq, uint32_t half, uint32_t position, float factor,
                                             uint32_t threads, float* cos_s, float* sin_s) {
  for (uint32_t i = threadIdx.x; i < half; i += threads) {
    const double angle = (double)position * freq[i];
    const double turns = rint(angle * 0.15915494309189535);
    double r = fma(-turns, 6.283185307179586, angle);  // 2 pi in two parts
    r = fma(-turns, 2.4492935982947064e-16, r);
    float sn, cs;
    sincosf((float)r, &sn, &cs);
    cos_s[i] = cs * factor;
    sin_s[i] = sn * factor;
  }
}

// Eight pairs' or four interleaved pairs' rotation, c their place in the table.  (Which
// product of a sum is rounded first is written out, so that the same form of rows gives
// the same bits in every kernel.  The form of single elements rounds the other product of a
// pair's second element first, as it always has.)
__device__ __forceinline__ void turn_interleaved(const float (&x)[8], float (&y)[8], const float* cos_s, const float* sin_s,
                                                 uint32_t c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float cs = cos_s[c + j], sn = sin_s[c + j];
    y[2 * j] = __builtin_fmaf(x[2 * j], cs, -(x[2 * j + 1] * sn));
    y[2 * j + 1] = __builtin_fmaf(x[2 * j + 1], cs, x[2 * j] * sn);
  }
}
__device__ __forceinline__ void turn_halves(const float (&x)[8], const float (&z)[8], float (&y)[8], float (&w)[8],
                                            const float* cos_s, const float* sin_s, uint32_t c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float cs = cos_s[c + j], sn = sin_s[c + j];
    y[j] = __builtin_fmaf(x[j], cs, -(z[j] * sn));
    w[j] = __builtin_fmaf(z[j], cs, x[j] * sn);
  }
}

// Work item `local` of one row of a tensor: 8 elements of a head (VEC) or one.
template <bool INTERLEAVED, bool VEC>
__device__ __forceinline__ void rotary_item(const RotaryTensor& t, const uint16_t* in, uint16_t* out, uint32_t local,
                                            uint32_t rd, const float* cos_s, const float* sin_s) {
  const uint32_t half = rd / 2;
  if constexpr (VEC) {
    const uint32_t per = t.head_dim / 8, head = local / per, e = (local - head * per) * 8;
    const size_t at = (size_t)head * t.head_dim + e;
    const uint32_t c = e - t.offset;  // element of the rotated part (wraps below it)
    if (e < t.offset || c >= rd) {
      if (out != in) *(u32x4*)(out + at) = *(const u32x4*)(in + at);
      return;
    }
    float x[8], y[8];
    if constexpr (INTERLEAVED) {
      unpack8(*(const u32x4*)(in + at), x);
      turn_interleaved(x, y, cos_s, sin_s, c / 2);
      *(u32x4*)(out + at) = pack8(y);
    } else {
      if (c >= half) return;  // its partner's item takes it
      float z[8], w[8];
      unpack8(*(const u32x4*)(in + at), x);
      unpack8(*(const u32x4*)(in + at + half), z);
      turn_halves(x, z, y, w, cos_s, sin_s, c);
      *(u32x4*)(out + at) = pack8(y);
      *(u32x4*)(out + at + half) = pack8(w);
    }
  } else {
    const uint32_t head = local / t.head_dim, e = local - head * t.head_dim;
    const size_t at = (size_t)head * t.head_dim + e;
    const uint32_t c = e - t.offset;
    if (e < t.offset || c >= rd) {
      if (out != in) out[at] = in[at];
      return;
    }
    // The first element of a pair takes its second along.
    if (INTERLEAVED ? c % 2 != 0 : c >= half) return;
    const uint32_t f = INTERLEAVED ? c / 2 : c, step = INTERLEAVED ? 1 : half;
    const float x = bf16_to_f32(in[at]), z = bf16_to_f32(in[at + step]);
    out[at] = f32_to_bf16(__builtin_fmaf(x, cos_s[f], -(z * sin_s[f])));
    out[at + step] = f32_to_bf16(__builtin_fmaf(x, sin_s[f], z * cos_s[f]));
  }
}

// The same item (VEC) in two steps, for a caller that forms its table meanwhile.
struct RotaryPiece {
  u32x4 x, z;  // z: the pairs' other elements
};
template <bool INTERLEAVED>
__device__ __forceinline__ RotaryPiece rotary_load(const RotaryTensor& t, const uint16_t* in, uint32_t local, uint32_t rd) {
  const uint32_t per = t.head_dim / 8, head = local / per, e = (local - head * per) * 8;
  const uint16_t* at = in + (size_t)head * t.head_dim + e;
  const uint32_t c = e - t.offset;
  const bool turned = e >= t.offset && c < rd;
  RotaryPiece p;
  p.x = *(const u32x4*)at;
  p.z = !INTERLEAVED && turned && c < rd / 2 ? *(const u32x4*)(at + rd / 2) : p.x;
  return p;
}
template <bool INTERLEAVED>
__device__ __forceinline__ void rotary_finish(const RotaryTensor& t, const RotaryPiece& p, bool copy, uint16_t* out,
                                              uint32_t local, uint32_t rd, const float* cos_s, const float* sin_s) {
  const uint32_t half = rd / 2;
  const uint32_t per = t.head_dim / 8, head = local / per, e = (local - head * per) * 8;
  const size_t at = (size_t)head * t.head_dim + e;
  const uint32_t c = e - t.offset;
  if (e < t.offset || c >= rd) {
    if (copy) *(u32x4*)(out + at) = p.x;
    return;
  }
  float x[8], y[8];
  unpack8(p.x, x);
  if constexpr (INTERLEAVED) {
    turn_interleaved(x, y, cos_s, sin_s, c / 2);
    *(u32x4*)(out + at) = pack8(y);
  } else {
    if (c >= half) return;
    float z[8], w[8];
    unpack8(p.z, z);
    turn_halves(x, z, y, w, cos_s, sin_s, c);
    *(u32x4*)(out + at) = pack8(y);
    *(u32x4*)(out + at + half) = pack8(w);
  }
}

}  // namespace qm
