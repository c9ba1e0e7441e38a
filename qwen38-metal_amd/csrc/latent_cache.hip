// The 8-bit cache of latent attention: rows written and read back, and the
// weights in the kernels' layouts.
//
// A row's layout and quantiser: latent_append.h.
#include <algorithm>

#include "latent.h"
#include "latent_append.h"
#include "latent_device.h"

namespace qm {
namespace {

constexpr int kWaves = 4;

template <int R>
__global__ __launch_bounds__(64 * kWaves) void latent_append_kernel(LatentAppendArgs a) {
  const uint32_t item = (blockIdx.x * kWaves + (threadIdx.x >> 6)) * R;
  if (item >= a.items) return;  // wave-uniform
  latent_append_rows<R>(a.rows, a.to, a.first + item, item, a.items, threadIdx.x & 63);
}

// A wave a row, 8 elements a lane.  8192 rows of 512 + 64 (4.8 MB in, 9.4 out): 4.2 us.
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

// One thread per element of `up`; elements of W_uk also go to `down`.  Once a layer:
// 128 heads of 256 x 512 take 70 us.
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

// One workgroup per head.  A row's squares are summed relative to its largest
// element's power of two, so that weights of any size keep their norm; one that
// passes fp32, or is no number, stays so (compared as bits).
__global__ __launch_bounds__(256) void latent_wnorm_kernel(LatentDims d, const uint16_t* down, float* wnorm) {
  __shared__ uint32_t top[256];
  const uint16_t* w = down + (size_t)blockIdx.x * d.rank_pad * d.nope_pad;
  uint32_t best = 0;
  for (uint32_t r = threadIdx.x; r < d.rank_pad; r += 256) {
    const uint16_t* row = w + (size_t)r * d.nope_pad;
    uint32_t most = 0;
    for (uint32_t k = 0; k < d.nope_pad; k += 8) {
      float x[8];
      latent_unpack8(*(const u32x4*)(row + k), x);
      most = max(most, latent_top(x));
    }
    const uint32_t e = min(max(most & 0x7F800000u, 0x01000000u), 0x7E000000u);
    const float scale = __uint_as_float(0x7F000000u - e);
    float s = 0.0f;
    for (uint32_t k = 0; k < d.nope_pad; k += 8) {
      float x[8];
      latent_unpack8(*(const u32x4*)(row + k), x);
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(x[i] * scale, x[i] * scale, s);
    }
    best = max(best, __float_as_uint(sqrtf(s) * __uint_as_float(e)) & 0x7FFFFFFFu);
  }
  top[threadIdx.x] = best;
  __syncthreads();
  for (uint32_t n = 128; n; n /= 2) {
    if (threadIdx.x < n) top[threadIdx.x] = max(top[threadIdx.x], top[threadIdx.x + n]);
    __syncthreads();
  }
  if (threadIdx.x == 0) wnorm[blockIdx.x] = __uint_as_float(top[0]) * 1.0001f;
}

template <class From>
hipError_t weights(const LatentDims& d, From from, uint16_t* down, uint16_t* up, hipStream_t st) {
  const uint32_t n = (d.nope_pad + d.v_pad) * d.rank_pad;
  hipLaunchKernelGGL(latent_weights_kernel<From>, dim3((n + 255) / 256, d.heads), dim3(256), 0, st, d, from, down, up);
  return hipGetLastError();
}

}  // namespace

constexpr uint32_t kMostRows = 1u << 22;  // of a launch, whose threads stay below 2^32

// A wave a row while the chip holds four waves a SIMD of them, then four rows a wave.
hipError_t launch_latent_append(const LatentAppendArgs& args, hipStream_t st) {
  constexpr int kMany = 4;
  LatentAppendArgs a = args;
  for (uint64_t r0 = 0; r0 < args.items; r0 += kMostRows) {
    a.rows.kv = args.rows.kv + r0 * (args.rows.rank + args.rows.rope);
    a.first = args.first + (uint32_t)r0;
    a.items = (uint32_t)std::min<uint64_t>(kMostRows, args.items - r0);
    if (a.items <= 4096)
      hipLaunchKernelGGL(latent_append_kernel<1>, dim3((a.items + kWaves - 1) / kWaves), dim3(64 * kWaves), 0, st, a);
    else
      hipLaunchKernelGGL(latent_append_kernel<kMany>, dim3((a.items + kWaves * kMany - 1) / (kWaves * kMany)),
                         dim3(64 * kWaves), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_latent_wnorm(const LatentDims& d, const uint16_t* down, float* wnorm, hipStream_t st) {
  hipLaunchKernelGGL(latent_wnorm_kernel, dim3(d.heads), dim3(256), 0, st, d, down, wnorm);
  return hipGetLastError();
}

hipError_t launch_latent_load(const LatentRows& rows, uint32_t rank, uint32_t rope, uint32_t rank_pad, uint32_t first,
                              uint32_t count, uint16_t* out, hipStream_t st) {
  for (uint64_t r0 = 0; r0 < count; r0 += kMostRows) {
    const uint32_t n = (uint32_t)std::min<uint64_t>(kMostRows, count - r0);
    hipLaunchKernelGGL(latent_load_kernel, dim3((n + kWaves - 1) / kWaves), dim3(64 * kWaves), 0, st, rows, rank, rope,
                       rank_pad, first + (uint32_t)r0, n, out + r0 * (rank + rope));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
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
