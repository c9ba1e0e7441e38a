// Rotary positions on a part of every head, out of place or in place.
//
// A pair (a, b) of a head's rotated part becomes
//   (a cos - b sin, b cos + a sin),  angle = position * freq[i],
// the pair being elements (i, i + rd/2) in the half layout and (2i, 2i + 1) in
// the interleaved one.  freq is formed on the host in fp64 (with the scaling
// for long contexts), the angle in fp64 and reduced modulo 2 pi there: at
// position 131072 an fp32 angle is off by up to 8e-3 rad.
//
// A block takes one row and a share of its work items.  Its threads build the
// row's table of sines and cosines (one fp64 angle per frequency, shared by all
// heads) in LDS, then each turns items of 16 bytes: 8 elements of a head, which
// hold 4 whole pairs of the interleaved layout; in the half layout an item of
// the first half takes its partner in the second along.  Items outside the
// rotated part are copied when the output is another buffer.  The general form
// takes single elements of any alignment.  Bound by HBM: 2048 rows of 64 heads of
// 192 and of one of 576, 105 MB in and out, take 21 us (5.0 TB/s).
#include "common.h"
#include "rotary.h"

#include <algorithm>

namespace qm {
namespace {

constexpr int kThreads = 256;

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

template <bool INTERLEAVED, bool VEC>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  __shared__ float cos_s[kRotaryMaxDim / 2], sin_s[kRotaryMaxDim / 2];
  const uint32_t row = a.row0 + blockIdx.x;
  const uint32_t rd = a.rotary_dim, half = rd / 2;
  for (uint32_t i = threadIdx.x; i < half; i += kThreads) {
    const uint32_t p = a.positions ? a.positions[row] : a.base + row;
    const double angle = (double)p * a.freq[i];
    const double turns = rint(angle * 0.15915494309189535);
    double r = fma(-turns, 6.283185307179586, angle);  // 2 pi in two parts
    r = fma(-turns, 2.4492935982947064e-16, r);
    float sn, cs;
    sincosf((float)r, &sn, &cs);
    cos_s[i] = cs * a.factor;
    sin_s[i] = sn * a.factor;
  }
  __syncthreads();

  for (uint32_t item = blockIdx.y * kThreads + threadIdx.x; item < a.items; item += gridDim.y * kThreads) {
    uint32_t k = 0;
    while (k + 1 < a.n && item >= a.t[k + 1].item_begin) ++k;
    const RotaryTensor& t = a.t[k];
    const uint32_t local = item - t.item_begin;
    const uint16_t* in = t.in + (size_t)row * t.in_stride;
    uint16_t* out = t.out + (size_t)row * t.out_stride;
    if constexpr (VEC) {
      const uint32_t per = t.head_dim / 8, head = local / per, e = (local - head * per) * 8;
      const size_t at = (size_t)head * t.head_dim + e;
      const uint32_t c = e - t.offset;  // element of the rotated part (wraps below it)
      if (e < t.offset || c >= rd) {
        if (out != in) *(u32x4*)(out + at) = *(const u32x4*)(in + at);
        continue;
      }
      float x[8], y[8];
      if constexpr (INTERLEAVED) {
        unpack8(*(const u32x4*)(in + at), x);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float cs = cos_s[c / 2 + j], sn = sin_s[c / 2 + j];
          y[2 * j] = x[2 * j] * cs - x[2 * j + 1] * sn;
          y[2 * j + 1] = x[2 * j + 1] * cs + x[2 * j] * sn;
        }
        *(u32x4*)(out + at) = pack8(y);
      } else {
        if (c >= half) continue;  // its partner's item takes it
        float z[8], w[8];
        unpack8(*(const u32x4*)(in + at), x);
        unpack8(*(const u32x4*)(in + at + half), z);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float cs = cos_s[c + j], sn = sin_s[c + j];
          y[j] = x[j] * cs - z[j] * sn;
          w[j] = z[j] * cs + x[j] * sn;
        }
        *(u32x4*)(out + at) = pack8(y);
        *(u32x4*)(out + at + half) = pack8(w);
      }
    } else {
      const uint32_t head = local / t.head_dim, e = local - head * t.head_dim;
      const size_t at = (size_t)head * t.head_dim + e;
      const uint32_t c = e - t.offset;
      if (e < t.offset || c >= rd) {
        if (out != in) out[at] = in[at];
        continue;
      }
      // The first element of a pair takes its second along.
      if (INTERLEAVED ? c % 2 != 0 : c >= half) continue;
      const uint32_t f = INTERLEAVED ? c / 2 : c, step = INTERLEAVED ? 1 : half;
      const float x = bf16_to_f32(in[at]), z = bf16_to_f32(in[at + step]);
      out[at] = f32_to_bf16(x * cos_s[f] - z * sin_s[f]);
      out[at + step] = f32_to_bf16(z * cos_s[f] + x * sin_s[f]);
    }
  }
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& args, uint32_t M, bool interleaved, bool vec, hipStream_t st) {
  RotaryArgs a = args;
  uint64_t items = 0;
  for (uint32_t k = 0; k < a.n; ++k) {
    a.t[k].item_begin = (uint32_t)items;
    items += (uint64_t)a.t[k].heads * a.t[k].head_dim / (vec ? 8 : 1);
  }
  a.items = (uint32_t)items;
  constexpr uint32_t kMaxRows = 1u << 23;  // a launch's threads stay below 2^32
  auto kernel = interleaved ? (vec ? rotary_kernel<true, true> : rotary_kernel<true, false>)
                            : (vec ? rotary_kernel<false, true> : rotary_kernel<false, false>);
  for (uint64_t r0 = 0; r0 < M; r0 += kMaxRows) {
    a.row0 = (uint32_t)r0;
    const uint32_t rows = (uint32_t)std::min<uint64_t>(kMaxRows, M - r0);
    // Blocks of a row: one for many rows, more where the rows alone leave CUs idle.
    const uint32_t most = (a.items + kThreads - 1) / kThreads;
    const uint32_t groups = std::max(1u, std::min(most, (1024u + rows - 1) / rows));
    hipLaunchKernelGGL(kernel, dim3(rows, groups), dim3(kThreads), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace qm
