// The 8-bit cache of latent attention: rows written and read back, and the
// weights in the kernels' layouts.
//
// A token's row is its latent (rank_pad codes) and the shared key (64 codes),
// each with one fp32 scale: s = max(absmax / 127, FLT_MIN), code = round half
// away(clamp(x / s, -127, 127)) with IEEE division, the quantiser of the Q8 KV
// cache (but that a part with a NaN or an infinity stands for NaN).  The latent may be RMS-normalised on its way (x rsqrt(mean x^2 + eps)
// w), in fp32: the projection's row is read once and nothing else is written
// but the 8 bits.
//
// A wave takes a row: 8 elements per lane of the latent (16 bytes in, 8 out)
// and 8 per lane of lanes 0..7 of the key.
#include <float.h>

#include <algorithm>

#include "common.h"
#include "latent.h"

namespace qm {
namespace {

constexpr int kWaves = 4;

__device__ __forceinline__ void unpack8(u32x4 v, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_to_f32(v[i] & 0xFFFFu);
    x[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
  }
}

// Quantises a wave's row held 8 elements per lane; returns the scale: NaN, with
// codes of 0, for a row that holds a NaN or an infinity.
__device__ __forceinline__ float quantise(const float (&x)[8], u32x2* codes) {
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

__global__ __launch_bounds__(64 * kWaves) void latent_append_kernel(LatentAppendArgs a) {
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t item = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (item >= a.items) return;  // wave-uniform
  const uint16_t* src = a.kv + (size_t)item * (a.rank + a.rope);
  const uint32_t e = 8 * lane;
  const u32x4 none = {0, 0, 0, 0};
  const u32x4 lat = e < a.rank ? *(const u32x4*)(src + e) : none;
  const u32x4 key = e < a.rope ? *(const u32x4*)(src + a.rank + e) : none;
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = a.norm && e < a.rank ? a.norm[e + i] : 1.0f;
  float x[8], k[8];
  unpack8(lat, x);
  unpack8(key, k);
  if (a.norm) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
    const float r = 1.0f / sqrtf(wave_allsum(ss) / (float)a.rank + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
  }
  u32x2 cx, ck;
  const float sx = quantise(x, &cx), sk = quantise(k, &ck);
  const LatentRows& to = a.seqs[a.decode ? item : 0];
  const size_t token = a.decode ? a.pos[item] : (size_t)a.pos[0] + item;
  int8_t* row = to.codes + token * (a.rank_pad + kLatentRope);
  if (e < a.rank_pad) *(u32x2*)(row + e) = cx;
  if (e < kLatentRope) *(u32x2*)(row + a.rank_pad + e) = ck;
  if (lane == 0) *(float2*)(to.scales + 2 * token) = float2{sx, sk};
}

__global__ __launch_bounds__(64 * kWaves) void latent_load_kernel(LatentRows rows, uint32_t rank, uint32_t rope,
                                                                  uint32_t rank_pad, uint32_t first, uint32_t count,
                                                                  uint16_t* out) {
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t item = blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (item >= count) return;
  const size_t token = (size_t)first + item;
  const int8_t* row = rows.codes + token * (rank_pad + kLatentRope);
  const float2 s = *(const float2*)(rows.scales + 2 * token);
  uint16_t* dst = out + (size_t)item * (rank + rope);
  const uint32_t e = 8 * lane;
  auto part = [&](const int8_t* from, float scale, uint16_t* to) __attribute__((always_inline)) {
    const u32x2 c = *(const u32x2*)from;
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = f32_to_bf16((float)(int8_t)(c[i / 4] >> (8 * (i % 4))) * scale);
    *(u32x4*)to = u32x4{h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16)};
  };
  if (e < rank) part(row + e, s.x, dst + e);
  if (e < rope) part(row + rank_pad + e, s.y, dst + rank + e);
}

// Element (head, output row n of [nope + v], latent element r) of kv_b.
struct FromBf16 {
  const uint16_t* w;
  __device__ uint16_t operator()(const LatentDims& d, uint32_t h, uint32_t n, uint32_t r) const {
    return w[((size_t)h * (d.nope + d.v) + n) * d.rank + r];
  }
};
struct FromQ4 {  // affine: q * scale + bias for each 64 elements, rounded to bf16 (half a step, as bf16 weights are)
  const uint32_t* w;
  const uint16_t* s;
  const uint16_t* b;
  __device__ uint16_t operator()(const LatentDims& d, uint32_t h, uint32_t n, uint32_t r) const {
    const size_t row = (size_t)h * (d.nope + d.v) + n;
    const uint32_t q = (w[row * (d.rank / 8) + r / 8] >> (4 * (r % 8))) & 15u;
    const size_t g = row * (d.rank / 64) + r / 64;
    return f32_to_bf16((float)q * bf16_to_f32(s[g]) + bf16_to_f32(b[g]));
  }
};

// One thread per element of `up`; elements of W_uk also go to `down`.
template <class From>
__global__ __launch_bounds__(256) void latent_weights_kernel(LatentDims d, From from, uint16_t* down, uint16_t* up) {
  const uint32_t h = blockIdx.y, rows = d.nope_pad + d.v_pad;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;  // up's element of the head
  if (i >= rows * d.rank_pad) return;
  const uint32_t n = i / d.rank_pad, r = i - n * d.rank_pad;
  const bool key = n < d.nope_pad;
  const uint32_t m = key ? n : n - d.nope_pad;  // row of its kind
  uint16_t v = 0;
  if (r < d.rank && m < (key ? d.nope : d.v)) v = from(d, h, key ? m : d.nope + m, r);
  up[(size_t)h * rows * d.rank_pad + i] = v;
  if (key) down[((size_t)h * d.rank_pad + r) * d.nope_pad + n] = v;
}

template <class From>
hipError_t weights(const LatentDims& d, From from, uint16_t* down, uint16_t* up, hipStream_t st) {
  const uint32_t n = (d.nope_pad + d.v_pad) * d.rank_pad;
  hipLaunchKernelGGL(latent_weights_kernel<From>, dim3((n + 255) / 256, d.heads), dim3(256), 0, st, d, from, down, up);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_latent_append(const LatentAppendArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(latent_append_kernel, dim3((a.items + kWaves - 1) / kWaves), dim3(64 * kWaves), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_latent_load(const LatentRows& rows, uint32_t rank, uint32_t rope, uint32_t rank_pad, uint32_t first,
                              uint32_t count, uint16_t* out, hipStream_t st) {
  hipLaunchKernelGGL(latent_load_kernel, dim3((count + kWaves - 1) / kWaves), dim3(64 * kWaves), 0, st, rows, rank,
                     rope, rank_pad, first, count, out);
  return hipGetLastError();
}

hipError_t launch_latent_weights(const LatentDims& d, const uint16_t* kv_b, uint16_t* down, uint16_t* up,
                                 hipStream_t st) {
  return weights(d, FromBf16{kv_b}, down, up, st);
}
hipError_t launch_latent_weights_q4(const LatentDims& d, const uint32_t* w, const uint16_t* s, const uint16_t* b,
                                    uint16_t* down, uint16_t* up, hipStream_t st) {
  return weights(d, FromQ4{w, s, b}, down, up, st);
}

}  // namespace qm
