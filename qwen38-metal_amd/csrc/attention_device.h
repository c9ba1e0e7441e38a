// Device code shared by the attention kernels over 8-bit and 4-bit KV caches.
#pragma once
#include <float.h>

#include "attention.h"
#include "common.h"

namespace qm {

constexpr float kLog2e = 1.4426950408889634f;

// Eight bf16 of a query/gate row starting at element d0, zero past the real
// dimension dr; `full` (dr == Dp) takes one 16-byte load.
__device__ __forceinline__ u32x4 load_bf16x8(const uint16_t* row, uint32_t d0, uint32_t dr, bool full) {
  if (full) return *(const u32x4*)(row + d0);
  uint32_t h[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = d0 + e < dr ? (uint32_t)row[d0 + e] : 0u;
  return u32x4{h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16)};
}

// Physical page of logical page p: pages materialised by this call are not
// in the device table until this call writes them.
__device__ __forceinline__ int32_t page_id(const AttnSeq& sq, uint32_t p) {
  return sq.new_page_count > 0 && (int32_t)p >= sq.new_page_first ? sq.new_page_id + ((int32_t)p - sq.new_page_first)
                                                                 : sq.pt[p];
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}

// Two fp32 values -> packed bf16 (round to nearest even, v_cvt_pk_bf16_f32).
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const bf16x2_t v = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ float bf16_lo_f32(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi_f32(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// Maximum over the four lanes l, l^16, l^32, l^48 (the kq lanes of one MFMA
// column) with the gfx950 row-swap permutes instead of LDS shuffles.
__device__ __forceinline__ float max4_across_kq(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  // fmaxf is v_max_f32 (one operation; the operands are never NaN), where a
  // compare and select would be two plus a VCC hazard wait.
  const float m = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The same sum.
__device__ __forceinline__ float sum4_across_kq(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float m = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Maximum over lanes l and l ^ 32 (the two halves of one 32-wide MFMA column).
__device__ __forceinline__ float max2_across_halves(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}

template <bool B>
struct BoolTag {
  static constexpr bool value = B;
};

// Sigmoid of a bf16 gate.  A bf16 (8 bits) times log2(e) cut to 16 bits is exact,
// and what the cut takes from the exponential goes into the Newton step of the
// reciprocal.  Over every bf16 gate from -87 up: at most 1.95 ulp, 0.250 rms,
// where expf and an IEEE division (sigmoid_f) have 1.98 and 0.252; a sigmoid
// below the smallest normal number is zero.  The limits, which pass NaN on,
// keep infinities out of the products.  A wave ends with up to 128 of these in
// a row, and a short prompt waits for that: 2 rows of 24 / 4 heads of 256 take
// 17.2 us a call, 23.6 with sigmoid_f and the integer form of f32_to_bf16.
__device__ __forceinline__ float gate_sigmoid(float x) {
  constexpr float kCut = 1.44268798828125f;
  constexpr float kRest = (float)((1.0 - 1.4426950408889634 / kCut) * 0.6931471805599453);
  const float t = __builtin_elementwise_maximum(__builtin_elementwise_minimum(x * -kCut, 127.0f), -126.0f);
  const float e = __builtin_amdgcn_exp2f(t), d = 1.0f + e, q = __builtin_amdgcn_rcpf(d);
  const float n = __builtin_fmaf(e * (t * kRest), q, __builtin_fmaf(-d, q, 1.0f));
  return __builtin_fmaf(n, q, q);
}

// Four outputs as bf16, and with the sigmoid of four bf16 gates.
__device__ __forceinline__ u32x2 bf16x4_of(floatx4 v) {
  return u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}
__device__ __forceinline__ u32x2 gated_bf16x4(floatx4 v, u32x2 gate) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i < 2 ? gate.x : gate.y;
    const float x = i & 1 ? bf16_hi_f32(w) : bf16_lo_f32(w);
    v[i] *= gate_sigmoid(x);
  }
  return bf16x4_of(v);
}

}  // namespace qm
