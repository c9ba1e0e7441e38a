// Device helpers of the latent attention kernels.
#pragma once
#include "common.h"

namespace qm {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));

// A buffer descriptor (uniform): reads beyond its bytes give zero.
__device__ __forceinline__ u32x4 latent_rsrc(const void* base, uint32_t bytes) {
  const uint64_t p = (uint64_t)base;
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)p),
               (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(p >> 32)) & 0xFFFFu,
               (uint32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}

// Builtins of the device pass only.
#if defined(__HIP_DEVICE_COMPILE__)
#define QM_LDS(T, p) ((__attribute__((address_space(3))) T*)(p))
// Buffer -> LDS copies: lane i's bytes at voff + soff land at lds + i * size (lds
// and soff uniform).  In asm, because the compiler lets every LDS read that
// follows the builtin wait for the copy (any LDS address may be the one it
// writes) and so ends the overlap; the waits are latent_wait_vmcnt's.  The copies
// have no register output, and the waits that the compiler counts for its own
// loads only become stricter by them.  s_nop: M0, and scalar registers that a vector
// instruction wrote, have to settle before a memory instruction reads them.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 among the clobbers
__device__ __forceinline__ uint32_t latent_lds_address(const void* lds) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);  // a generic LDS address' lower half is the offset
}
__device__ __forceinline__ void latent_dma16(u32x4 r, void* lds, uint32_t voff, uint32_t soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :: "s"(latent_lds_address(lds)), "v"(voff), "s"(r), "s"(__builtin_amdgcn_readfirstlane(soff)) : "memory", "m0");
}
__device__ __forceinline__ void latent_dma4(u32x4 r, void* lds, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :: "s"(latent_lds_address(lds)), "v"(voff), "s"(r) : "memory", "m0");
}
#pragma clang diagnostic pop
// Transposing read of bytes: each 16 lanes read 8 rows of 16 bytes (lanes 2t
// and 2t + 1 give the address of row t's two halves) and lane i receives byte i
// of the 8 rows.
__device__ __forceinline__ u32x2 lds_read_tr8(const uint8_t* lds) {
  typedef int intx2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(QM_LDS(intx2, lds)));
}
__device__ __forceinline__ intx16 mfma32x32x32_i8(u32x4 a, u32x4 b, intx16 c) {
  return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(intx4, a), __builtin_bit_cast(intx4, b), c, 0, 0, 0);
}
#undef QM_LDS
#else
__device__ void latent_dma16(u32x4, void*, uint32_t, uint32_t);
__device__ void latent_dma4(u32x4, void*, uint32_t);
__device__ u32x2 lds_read_tr8(const uint8_t*);
__device__ intx16 mfma32x32x32_i8(u32x4, u32x4, intx16);
#endif

// s_waitcnt vmcnt(n) (gfx9 encoding; expcnt and lgkmcnt left at their maxima).
template <int N>
__device__ __forceinline__ void latent_wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 0xF) | ((N >> 4) << 14));
  __asm__ volatile("" ::: "memory");
}
// s_waitcnt lgkmcnt(0): this wave's LDS reads have returned.
__device__ __forceinline__ void latent_wait_lds() {
  __asm__ volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);
  __asm__ volatile("" ::: "memory");
}

// Two fp32 values -> packed fp16 (round to nearest even, v_cvt_pk_f16_f32).
typedef _Float16 latent_halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 latent_halfx4 __attribute__((ext_vector_type(4)));
typedef _Float16 latent_halfx8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ uint32_t to_f16x2(float lo, float hi) {
  const latent_halfx2 v = {(_Float16)lo, (_Float16)hi};
  return __builtin_bit_cast(uint32_t, v);
}
// 8 signed bytes -> 8 fp16, exact, in the order 0, 2, 1, 3, 4, 6, 5, 7: 0x6400 | u
// is the fp16 1024 + u, so each pair takes one permute and one packed subtraction.
__device__ __forceinline__ u32x4 bytes_to_f16(u32x2 w) {
  const latent_halfx4 bias = {(_Float16)1152.0f, (_Float16)1152.0f, (_Float16)1152.0f, (_Float16)1152.0f};
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t u = w[i] ^ 0x80808080u;
    const u32x2 biased = {perm_b32(u, 0x64646464u, 0x00060004u), perm_b32(u, 0x64646464u, 0x00070005u)};
    const u32x2 v = __builtin_bit_cast(u32x2, __builtin_bit_cast(latent_halfx4, biased) - bias);
    r[2 * i] = v.x;
    r[2 * i + 1] = v.y;
  }
  return r;
}
__device__ __forceinline__ floatx16 mfma32x32x16_f16(u32x4 a, u32x4 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(latent_halfx8, a),
                                                __builtin_bit_cast(latent_halfx8, b), c, 0, 0, 0);
}

// Two fp32 values -> packed bf16 (round to nearest even, v_cvt_pk_bf16_f32).
typedef __bf16 latent_bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t to_bf16x2(float lo, float hi) {
  const latent_bf16x2 v = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(uint32_t, v);
}
// The upper lanes' `a` and the lower lanes' `b` change places.
__device__ __forceinline__ void swap_halves(uint32_t& a, uint32_t& b) {
  const auto p = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = p[0], b = p[1];
}
// Maximum of lanes l and l ^ 32, and their sum.
__device__ __forceinline__ float halves_max(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

}  // namespace qm
