// Rows into the paged KV caches without attention, keys and queries rotated on the
// way, and rows read back.
//
// A key's rotated pair is (a cos - b sin, b cos + a sin) as in rotary.hip, but in
// fp64, rounded once to fp32: its code is decided by what lies on either side of a
// border, and what 4 or 8 bits make of a key then depends on the key alone.  Sine
// and cosine are their Taylor series on [-pi/4, pi/4] (error below 1e-13).  Queries
// take rotary.hip's own arithmetic, and so its bits.
//
// 4 bits, per group of 64 elements of a (token, KV head):
//   s = bf16(max((max - min) / 15, FLT_MIN)),  m = bf16(min + 8 s),
//   c = round half to even(clamp((x - m) / s, -8, 7)),  x ~ s c + m.
// Both roundings to bf16 happen before the codes are chosen, so a code makes up for
// them; m lies in the middle of the values, where bf16 costs least.  A group with a
// NaN or an infinity stands for NaN (s and m).  8 bits: as the attention kernels'
// own append.
//
// A workgroup takes a (page, KV head) of one sequence: the lanes of a row of 16
// hold a group, 4 elements each, so its statistics are DPP steps within the row;
// codes meet in LDS in the page's layout and leave in 8-byte pieces.  Where the
// call fills only part of a page the words that several tokens share keep the other
// tokens' nibbles.  Further workgroups of the launch rotate the queries.
#include <float.h>

#include <algorithm>

#include "kv_append.h"
#include "kv_quant.h"
#include "q4kv.h"
#include "rotary_device.h"

namespace qm {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// Four elements of a row from element d on, zero past dr.
template <bool VEC>
__device__ __forceinline__ void load4(const float* row, uint32_t d, uint32_t dr, float (&x)[4]) {
  if constexpr (VEC) {
    const floatx4 w = d < dr ? *(const floatx4*)(row + d) : floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = w[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = d + e < dr ? row[d + e] : 0.0f;
  }
}
template <bool VEC>
__device__ __forceinline__ void load4(const uint16_t* row, uint32_t d, uint32_t dr, float (&x)[4]) {
  if constexpr (VEC) {
    const u32x2 w = d < dr ? *(const u32x2*)(row + d) : u32x2{0u, 0u};
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = bf16_to_f32(e & 1 ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = d + e < dr ? bf16_to_f32(row[d + e]) : 0.0f;
  }
}

// Where element d's partner of the rotation lies, the frequency of the pair, and
// whether d is its first element.
struct Pair {
  uint32_t partner, freq;
  bool turned, first;
};
template <bool INTERLEAVED>
__device__ __forceinline__ Pair pair_of(uint32_t d, uint32_t offset, uint32_t rd) {
  const uint32_t c = d - offset, half = rd / 2;  // wraps below the offset
  if (d < offset || c >= rd) return Pair{d, 0, false, false};
  if (INTERLEAVED) return Pair{c & 1 ? d - 1 : d + 1, c / 2, true, (c & 1) == 0};
  return c < half ? Pair{d + half, c, true, true} : Pair{d - half, c - half, true, false};
}

// T: uint16_t (bf16 rows) or float (rows prepared by the caller, not rotated).
template <int BITS, class T, bool INTERLEAVED, bool VEC, bool QVEC>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(KvAppendArgs a) {
  // Sines and cosines of a page's tokens (keys) or of a row (queries).
  __shared__ __attribute__((aligned(16))) double cos_d[16][kRotaryMaxDim / 2], sin_d[16][kRotaryMaxDim / 2];
  __shared__ __attribute__((aligned(16))) uint8_t k_img[8 * 256];  // 4 bits: the page's K part
  __shared__ __attribute__((aligned(16))) uint8_t v_codes[16 * 256];  // 4 bits: [token][d]; 8 bits: [d][token]
  const uint32_t tid = threadIdx.x;

  if (blockIdx.x >= a.units) {  // queries: a row, or a share of its items
    const uint32_t x = blockIdx.x - a.units, row = a.row0 + x / a.q_groups;
    uint32_t b = 0;
    while (b + 1 < a.n_seqs && row >= a.seqs[b + 1].row0) ++b;
    // (a sequence without rows shares its row0 with the next one, so b has some)
    const uint32_t position = a.positions ? a.positions[row] : a.seqs[b].start + (row - a.seqs[b].row0);
    float *cos_s = (float*)cos_d, *sin_s = (float*)sin_d;
    rotary_table(a.freq, a.rotary_dim / 2, position, a.factor, kThreads, cos_s, sin_s);
    __syncthreads();
    for (uint32_t item = x % a.q_groups * kThreads + tid; item < a.q_items; item += a.q_groups * kThreads)
      rotary_item<INTERLEAVED, QVEC>(a.q, a.q.in + (size_t)row * a.q.in_stride, a.q.out + (size_t)row * a.q.out_stride,
                                     item, a.rotary_dim, cos_s, sin_s);
    return;
  }

  uint32_t b = 0;
  while (b + 1 < a.n_seqs && blockIdx.x >= a.seqs[b + 1].unit_begin) ++b;
  const KvAppendSeq& sq = a.seqs[b];
  const uint32_t KVH = a.kv_heads, D = a.head_dim, Dp = a.head_dim_pad, G = Dp / 64;
  const uint32_t u = blockIdx.x - sq.unit_begin;
  const uint32_t page = sq.start / 16 + u / KVH, kvh = u % KVH;
  // Slots lo .. hi - 1 of the page are new; slot s is row `base + s` of the call.
  const uint32_t lo = max(sq.start, 16 * page) - 16 * page, hi = min(sq.start + sq.rows, 16 * page + 16) - 16 * page;
  const uint32_t base = sq.row0 + 16 * page - sq.start;  // (wraps where the page begins before the rows)
  const bool fresh = sq.new_page_count > 0 && (int32_t)page >= sq.new_page_first;
  const int32_t phys = fresh ? sq.new_page_id + ((int32_t)page - sq.new_page_first) : sq.p.pt[page];
  if (fresh && kvh == 0 && tid == 0) sq.p.pt[page] = phys;
  const size_t block = (size_t)phys * KVH + kvh;

  // Every load first: the wave's tokens, 4 / G at a time.
  const int lane = tid & 63, wave = tid >> 6;
  const uint32_t row16 = lane >> 4, i16 = lane & 15;
  const uint32_t g = row16 % G, d0 = 64 * g + 4 * i16;
  constexpr int kMaxPass = 4;
  constexpr bool kTurns = sizeof(T) == 2;
  float kx[kMaxPass][4], kp[kMaxPass][4], vx[kMaxPass][4];
#pragma unroll
  for (int p = 0; p < kMaxPass; ++p) {
    if (p >= (int)G) break;
    const uint32_t slot = (p * kWaves + wave) * (4 / G) + row16 / G;
    const size_t row = base + min(max(slot, lo), hi - 1);
    const T* kr = (const T*)a.k + row * a.k_stride + (size_t)kvh * D;
    load4<VEC>(kr, d0, D, kx[p]);
    load4<VEC>((const T*)a.v + row * a.v_stride + (size_t)kvh * D, d0, D, vx[p]);
    if constexpr (!kTurns) {
    } else if constexpr (VEC && !INTERLEAVED) {
      const Pair pr = pair_of<false>(d0, a.offset, a.rotary_dim);
      load4<true>(kr, pr.partner, D, kp[p]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Pair pr = pair_of<INTERLEAVED>(d0 + e, a.offset, a.rotary_dim);
        kp[p][e] = VEC ? kx[p][e ^ 1] : pr.turned && d0 + e < D ? bf16_to_f32(kr[pr.partner]) : 0.0f;
      }
    }
  }
  if (kTurns && a.rotary_dim) {
    const uint32_t half = a.rotary_dim / 2;
    for (uint32_t i = tid; i < (hi - lo) * half; i += kThreads) {
      const uint32_t slot = lo + i / half, f = i % half;
      const uint32_t position = a.positions ? a.positions[base + slot] : 16 * page + slot;
      double sn, cs;
      sincos_f64((double)position * a.freq[f], &sn, &cs);
      cos_d[slot][f] = cs * a.factor;
      sin_d[slot][f] = sn * a.factor;
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < kMaxPass; ++p) {
      if (p >= (int)G) break;
      const uint32_t slot = min(max((p * kWaves + wave) * (4 / G) + row16 / G, lo), hi - 1);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Pair pr = pair_of<INTERLEAVED>(d0 + e, a.offset, a.rotary_dim);
        if (!pr.turned) continue;
        const double x = kx[p][e], y = kp[p][e];
        kx[p][e] = (float)(x * cos_d[slot][pr.freq] + (pr.first ? -y : y) * sin_d[slot][pr.freq]);
      }
    }
  }

  uint32_t* scales = (uint32_t*)(sq.p.k + block * q4kv_block_bytes(Dp) + q4kv_scale_bytes(Dp));
#pragma unroll
  for (int p = 0; p < kMaxPass; ++p) {
    if (p >= (int)G) break;
    const uint32_t slot = (p * kWaves + wave) * (4 / G) + row16 / G;
    const bool mine = slot >= lo && slot < hi;
    if constexpr (BITS == 4) {
      int kc[4], vc[4];
      const uint32_t kw = q4kv_group(kx[p], d0, D, kc), vw = q4kv_group(vx[p], d0, D, vc);
      // Two lanes hold a K word.
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) w |= (uint32_t)(kc[e] + 8) << q4kv_k_bit((d0 + e) % 8);
      w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0xB1, 0xF, 0xF, false);
      if (mine) {
        if ((lane & 1) == 0) *(uint32_t*)(k_img + q4kv_k_word(Dp, slot, d0)) = w;
        *(uint32_t*)(v_codes + slot * Dp + d0) =
            (vc[0] + 8) | (vc[1] + 8) << 8 | (vc[2] + 8) << 16 | (vc[3] + 8) << 24;
        if (i16 == 0) {
          scales[q4kv_scale_word(Dp, 0, g, slot)] = kw;
          scales[q4kv_scale_word(Dp, 1, g, slot)] = vw;
        }
      }
    } else {
      int8_t kq[4], vq[4];
      const float ks = q8_rows_quant(kx[p], G, kq), vs = q8_rows_quant(vx[p], G, vq);
      if (mine) {
        *(uint32_t*)(sq.p.k + (block * 16 + slot) * Dp + d0) = pack_q8x4(kq);
#pragma unroll
        for (int e = 0; e < 4; ++e) v_codes[(d0 + e) * 16 + slot] = (uint8_t)vq[e];
        if (i16 == 0 && g == 0) {
          sq.p.ks[block * 16 + slot] = ks;
          sq.p.vs[block * 16 + slot] = vs;
        }
      }
    }
  }
  __syncthreads();

  if constexpr (BITS == 4) {
    if (tid < Dp) {  // 8-byte unit tid of the K part and of the V part
      const uint32_t l = Dp == 64 ? tid : tid % 128 / 2;
      uint8_t* kv = sq.p.k + block * q4kv_block_bytes(Dp);
      if ((l & 15) >= lo && (l & 15) < hi) *(u32x2*)(kv + 8 * tid) = *(const u32x2*)(k_img + 8 * tid);
      const uint32_t t0 = 4 * (l >> 4), d = 64 * (Dp == 64 ? 0 : 2 * (tid / 128) + tid % 2) + (l & 15);
      if (t0 < hi && t0 + 4 > lo) {
        u32x2* at = (u32x2*)(kv + q4kv_v_bytes(Dp) + 8 * tid);
        const bool whole = lo <= t0 && hi >= t0 + 4;
        u32x2 w = {0u, 0u};
        if (!whole) w = *at;
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
          if (t0 + r < lo || t0 + r >= hi) continue;
#pragma unroll
          for (uint32_t db = 0; db < 4; ++db) {
            const uint32_t bit = q4kv_v_bit(r, 16 * db), c = v_codes[(t0 + r) * Dp + d + 16 * db];
            w[db / 2] = (w[db / 2] & ~(15u << bit)) | c << bit;
          }
        }
        *at = w;
      }
    }
  } else if (tid < Dp) {
    uint8_t* at = sq.p.v + (block * Dp + tid) * 16;
    if (lo == 0 && hi == 16) {
      *(u32x4*)at = *(const u32x4*)(v_codes + 16 * tid);
    } else {
      for (uint32_t s = lo; s < hi; ++s) at[s] = v_codes[16 * tid + s];
    }
  }
}

// Reads back: a workgroup a (page, KV head), a thread four elements of a token.
template <int BITS>
__global__ __launch_bounds__(kThreads) void kv_load_kernel(KvLoadArgs a) {
  const uint32_t KVH = a.kv_heads, D = a.head_dim, Dp = a.head_dim_pad;
  const uint32_t page = a.first / 16 + blockIdx.x / KVH, kvh = blockIdx.x % KVH;
  const size_t block = (size_t)a.p.pt[page] * KVH + kvh;
  const uint32_t quads = Dp / 4;
  for (uint32_t i = threadIdx.x; i < 16 * quads; i += kThreads) {
    const uint32_t slot = i / quads, d0 = i % quads * 4;
    const uint32_t token = 16 * page + slot;
    if (token < a.first || token >= a.first + a.count || d0 >= D) continue;
    float k[4], v[4];
    if constexpr (BITS == 4) {
      const uint8_t* kv = a.p.k + block * q4kv_block_bytes(Dp);
      const uint32_t* scales = (const uint32_t*)(kv + q4kv_scale_bytes(Dp));
      const uint32_t kw = scales[q4kv_scale_word(Dp, 0, d0 / 64, slot)], vw = scales[q4kv_scale_word(Dp, 1, d0 / 64, slot)];
      const uint32_t kc = *(const uint32_t*)(kv + q4kv_k_word(Dp, slot, d0));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t vc = *(const uint32_t*)(kv + q4kv_v_bytes(Dp) + q4kv_v_word(Dp, slot, d0 + e));
        k[e] = q4kv_value((int)(kc >> q4kv_k_bit(d0 + e) & 15) - 8, kw);
        v[e] = q4kv_value((int)(vc >> q4kv_v_bit(slot, d0 + e) & 15) - 8, vw);
      }
    } else {
      const float ks = a.p.ks[block * 16 + slot], vs = a.p.vs[block * 16 + slot];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        k[e] = (float)(int8_t)a.p.k[(block * 16 + slot) * Dp + d0 + e] * ks;
        v[e] = (float)(int8_t)a.p.v[(block * Dp + d0 + e) * 16 + slot] * vs;
      }
    }
    const size_t at = ((size_t)(token - a.first) * KVH + kvh) * D + d0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (d0 + e >= D) break;
      if (a.k) a.k[at + e] = f32_to_bf16(k[e]);
      if (a.v) a.v[at + e] = f32_to_bf16(v[e]);
    }
  }
}

template <int BITS, bool INTERLEAVED>
void launch_append(const KvAppendArgs& a, bool vec, bool qvec, uint32_t grid, hipStream_t st) {
  auto kernel = vec ? (qvec ? kv_append_kernel<BITS, uint16_t, INTERLEAVED, true, true>
                            : kv_append_kernel<BITS, uint16_t, INTERLEAVED, true, false>)
                    : (qvec ? kv_append_kernel<BITS, uint16_t, INTERLEAVED, false, true>
                            : kv_append_kernel<BITS, uint16_t, INTERLEAVED, false, false>);
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), 0, st, a);
}

// Gives every sequence its workgroups; returns how many there are.
uint64_t plan_units(KvAppendArgs* a) {
  uint64_t units = 0;
  a->rows = 0;
  a->row0 = a->seqs[0].row0;
  for (uint32_t b = 0; b < a->n_seqs; ++b) {
    KvAppendSeq& s = a->seqs[b];
    s.unit_begin = (uint32_t)units;
    if (s.rows) units += (uint64_t)((s.start + s.rows - 1) / 16 - s.start / 16 + 1) * a->kv_heads;
    a->rows += s.rows;
  }
  a->units = (uint32_t)units;
  return units;
}

}  // namespace

hipError_t launch_kv_append(const KvAppendArgs& args, uint32_t bits, bool interleaved, bool vec, bool qvec,
                            hipStream_t st) {
  KvAppendArgs a = args;
  uint64_t grid = plan_units(&a);
  if (a.rows == 0) return hipSuccess;
  if (a.q.in) {
    a.q_items = a.q.heads * a.q.head_dim / (qvec ? 8 : 1);
    const uint32_t most = (a.q_items + kThreads - 1) / kThreads;
    a.q_groups = std::max(1u, std::min(most, (1024u + a.rows - 1) / a.rows));
    grid += (uint64_t)a.rows * a.q_groups;
  }
  if (grid > 0xFFFFFFFFull / kThreads) return hipErrorInvalidValue;
  if (bits == 4)
    interleaved ? launch_append<4, true>(a, vec, qvec, (uint32_t)grid, st)
                : launch_append<4, false>(a, vec, qvec, (uint32_t)grid, st);
  else
    interleaved ? launch_append<8, true>(a, vec, qvec, (uint32_t)grid, st)
                : launch_append<8, false>(a, vec, qvec, (uint32_t)grid, st);
  return hipGetLastError();
}

hipError_t launch_q4kv_append_f32(const KvAppendArgs& args, bool vec, hipStream_t st) {
  KvAppendArgs a = args;
  const uint64_t grid = plan_units(&a);
  if (a.rows == 0) return hipSuccess;
  if (grid > 0xFFFFFFFFull / kThreads) return hipErrorInvalidValue;
  auto kernel = vec ? kv_append_kernel<4, float, false, true, false> : kv_append_kernel<4, float, false, false, false>;
  hipLaunchKernelGGL(kernel, dim3((uint32_t)grid), dim3(kThreads), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_kv_load(const KvLoadArgs& a, uint32_t bits, hipStream_t st) {
  const uint64_t units = (uint64_t)((a.first + (uint64_t)a.count - 1) / 16 - a.first / 16 + 1) * a.kv_heads;
  if (a.count == 0 || units > 0xFFFFFFFFull / kThreads) return hipErrorInvalidValue;
  auto kernel = bits == 4 ? kv_load_kernel<4> : kv_load_kernel<8>;
  hipLaunchKernelGGL(kernel, dim3((uint32_t)units), dim3(kThreads), 0, st, a);
  return hipGetLastError();
}

}  // namespace qm
