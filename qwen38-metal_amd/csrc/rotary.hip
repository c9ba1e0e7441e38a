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
#include "rotary_device.h"

#include <algorithm>

namespace qm {
namespace {

constexpr int kThreads = 256;

template <bool INTERLEAVED, bool VEC>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  __shared__ float cos_s[kRotaryMaxDim / 2], sin_s[kRotaryMaxDim / 2];
  const uint32_t row = a.row0 + blockIdx.x;
  rotary_table(a.freq, a.rotary_dim / 2, a.positions ? a.positions[row] : a.base + row, a.factor, kThreads, cos_s,
               sin_s);
  __syncthreads();

  for (uint32_t item = blockIdx.y * kThreads + threadIdx.x; item < a.items; item += gridDim.y * kThreads) {
    uint32_t k = 0;
    while (k + 1 < a.n && item >= a.t[k + 1].item_begin) ++k;
    const RotaryTensor& t = a.t[k];
    rotary_item<INTERLEAVED, VEC>(t, t.in + (size_t)row * t.in_stride, t.out + (size_t)row * t.out_stride,
                                  item - t.item_begin, a.rotary_dim, cos_s, sin_s);
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
