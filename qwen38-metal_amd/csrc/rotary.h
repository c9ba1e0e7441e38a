// Launch interface of the stand-alone rotary positions (rotary.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qm {

constexpr uint32_t kRotaryMaxDim = 256;
constexpr uint32_t kRotaryMaxTensors = 4;

struct RotaryTensor {
  const uint16_t* in;
  uint16_t* out;
  uint64_t in_stride;   // elements between rows
  uint64_t out_stride;
  uint32_t heads;
  uint32_t head_dim;    // elements between heads
  uint32_t offset;      // first rotated element of a head
  uint32_t item_begin;  // filled by the launcher
};

struct RotaryArgs {
  double freq[kRotaryMaxDim / 2];  // radians per position
  RotaryTensor t[kRotaryMaxTensors];
  const uint32_t* positions;  // [M], or null: base + row
  uint32_t base;
  uint32_t row0;
  uint32_t n;           // tensors
  uint32_t items;       // work items of a row
  uint32_t rotary_dim;
  float factor;         // of sine and cosine
};

// Rows row0 = 0 .. M - 1.  `vec`: every row, head and part starts on 16 bytes
// and the rotated part is whole 8-element pieces (of each half).
hipError_t launch_rotary(const RotaryArgs& a, uint32_t M, bool interleaved, bool vec, hipStream_t st);

}  // namespace qm
