// Rows into the paged KV caches without attention, keys and queries rotated on the
// way, and rows read back.
//
// A key's rotated pair is (a cos - b sin, b cos + a sin) as in rotary.hip, but in
// fp64, rounded once to fp32: its code is decided by what lies on either side of a
// border, and what 4 or 8 bits make of a key then depends on the key alone.  Sine
// and cosine are their Taylor series on [-pi/4, pi/4] (error below 1e-13).  Queries
// take rotary.hip's own arithmetic, and so the bits that it gives for the same rows.
//
// 4 bits, per group of 64 elements of a (token, KV head):
//   s = bf16(max((max - min) / 15, FLT_MIN)),  m = bf16(min + 8 s),
//   c = round half to even(clamp((x - m) / s, -8, 7)),  x ~ s c + m.
// Both roundings to bf16 happen before the codes are chosen, so a code makes up for
// them; m lies in the middle of the values, where bf16 costs least.  A group with a
// NaN or an infinity stands for NaN (s and m).  8 bits: as the attention kernels'
// own append.
//
// A workgroup of 4 Dp threads takes a page of one sequence and one KV head of it, or
// several where the call is long: they share its sines and cosines, which cost as much
// as a head's codes.  A thread holds 4 elements of a key and of a value, a lane row of
// 16 a group, so its statistics are DPP steps within the row; codes meet in LDS in the
// page's layout and leave in 8-byte pieces.  Where the call fills only part of a page
// the words that several tokens share keep the other tokens' nibbles.  Further
// workgroups of the launch rotate the queries.
//
// Bound by memory where queries are rotated too (8192 rows of 64 / 8 heads of 128: 67 us,
// 311 MB at 4.6 TB/s), else by its vector instructions (16384 rows of 8 / 8 heads: 72 us
// for 153 MB).  Registers are held to 64, so that two workgroups share a CU at Dp = 256 (84
// us for 8192 rows of 24 / 4 heads of 256, against 97 with 82 registers).  One token: 5 us,
// the chain of its page id, its rows, its table and its codes.
#include <float.h>

#include <algorithm>

#include "attention_device.h"
#include "kv_append.h"
#include "kv_quant.h"
#include "q4kv.h"
#include "rotary_device.h"

namespace qm {
namespace {

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
__global__ __launch_bounds__(1024, VEC ? 8 : 4) void kv_append_kernel(KvAppendArgs a) {
  // Sines and cosines: fp64, of a page's tokens (keys), or fp32, of a row (queries).
  extern __shared__ __attribute__((aligned(16))) uint8_t table[];
  __shared__ __attribute__((aligned(16))) uint8_t k_img[8 * 256];  // 4 bits: the page's K part
  // [d][token], rows of whole words (4 bits: 20 bytes, which spreads the writes of a lane
  // row over the banks).
  constexpr uint32_t kVRow = BITS == 4 ? 20 : 16;
  __shared__ __attribute__((aligned(16))) uint8_t v_codes[kVRow * 256];
  const uint32_t tid = threadIdx.x, threads = 4 * a.head_dim_pad, half = a.rotary_dim / 2;
  const int lane = tid & 63, wave = tid >> 6;
  // The sequence of a workgroup or row: the last that starts at or below it (one without
  // any shares its start with the next).  A lane looks at each.
  auto sequence_of = [&](uint32_t x, auto start) __attribute__((always_inline)) {
    if (a.n_seqs == 1) return 0;
    return __builtin_popcountll(__builtin_amdgcn_ballot_w64((uint32_t)lane < a.n_seqs && x >= start(a.seqs[lane % kMaxAppendSeqs]))) - 1;
  };

  if (blockIdx.x >= a.units) {  // queries: a row, or a share of its items
    const uint32_t x = blockIdx.x - a.units, row = a.row0 + x / a.q_groups, step = a.q_groups * threads;
    uint32_t item = x % a.q_groups * threads + tid;
    const uint16_t* in = a.q.in + (size_t)row * a.q.in_stride;
    uint16_t* out = a.q.out + (size_t)row * a.q.out_stride;
    RotaryPiece next{};  // on its way while the table is formed
    if (QVEC && item < a.q_items) next = rotary_load<INTERLEAVED>(a.q, in, item, a.rotary_dim);
    const int b = sequence_of(row, [](const KvAppendSeq& s) { return s.row0; });
    const uint32_t position = a.positions ? a.positions[row] : a.seqs[b].start + (row - a.seqs[b].row0);
    float *cos_s = (float*)table, *sin_s = cos_s + half;
    rotary_table(a.freq, half, position, a.factor, threads, cos_s, sin_s);
    __syncthreads();
    for (; item < a.q_items; item += step) {
      if constexpr (QVEC) {
        const RotaryPiece p = next;
        if (item + step < a.q_items) next = rotary_load<INTERLEAVED>(a.q, in, item + step, a.rotary_dim);
        rotary_finish<INTERLEAVED>(a.q, p, out != in, out, item, a.rotary_dim, cos_s, sin_s);
      } else {
        rotary_item<INTERLEAVED, false>(a.q, in, out, item, a.rotary_dim, cos_s, sin_s);
      }
    }
    return;
  }

  const KvAppendSeq& sq = a.seqs[sequence_of(blockIdx.x, [](const KvAppendSeq& s) { return s.unit_begin; })];
  const uint32_t KVH = a.kv_heads, D = a.head_dim, Dp = a.head_dim_pad, G = Dp / 64;
  const uint32_t u = blockIdx.x - sq.unit_begin, shares = (KVH + a.share - 1) / a.share;
  const uint32_t page = sq.start / 16 + u / shares, kvh0 = u % shares * a.share, kvh1 = min(kvh0 + a.share, KVH);
  // Slots lo .. hi - 1 of the page are new; slot s is row `base + s` of the call.
  const uint32_t lo = max(sq.start, 16 * page) - 16 * page, hi = min(sq.start + sq.rows, 16 * page + 16) - 16 * page;
  const uint32_t base = sq.row0 + 16 * page - sq.start;  // (wraps where the page begins before the rows)
  const bool fresh = sq.new_page_count > 0 && (int32_t)page >= sq.new_page_first;
  const int32_t phys = fresh ? sq.new_page_id + ((int32_t)page - sq.new_page_first) : sq.p.pt[page];
  if (fresh && kvh0 == 0 && tid == 0) sq.p.pt[page] = phys;

  // The wave's 4 / G tokens: slots of the page, and the rows that it reads.
  const uint32_t row16 = lane >> 4, i16 = lane & 15;
  const uint32_t g = row16 % G, d0 = 64 * g + 4 * i16, slot = wave * (4 / G) + row16 / G;
  const bool mine = slot >= lo && slot < hi;
  const uint32_t there = min(max(slot, lo), hi - 1);
  constexpr bool kTurns = sizeof(T) == 2;
  float x[2][4], kp[4];  // the key, the value; the key's pairs' other elements
  auto load_head = [&](uint32_t kvh) __attribute__((always_inline)) {
    const size_t row = base + there;
    const T* kr = (const T*)a.k + row * a.k_stride + (size_t)kvh * D;
    load4<VEC>(kr, d0, D, x[0]);
    load4<VEC>((const T*)a.v + row * a.v_stride + (size_t)kvh * D, d0, D, x[1]);
    if constexpr (!kTurns) {
    } else if constexpr (VEC && !INTERLEAVED) {
      const Pair pr = pair_of<false>(d0, a.offset, a.rotary_dim);
      load4<true>(kr, pr.partner, D, kp);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const Pair pr = pair_of<INTERLEAVED>(d0 + e, a.offset, a.rotary_dim);
        kp[e] = VEC ? x[0][e ^ 1] : pr.turned && d0 + e < D ? bf16_to_f32(kr[pr.partner]) : 0.0f;
      }
    }
  };
  load_head(kvh0);
  // 4 bits: thread tid's 8-byte unit of the K part and of the V part.  Where other tokens
  // share the V unit's words they keep their nibbles.
  const uint32_t ul = Dp == 64 ? tid : tid % 128 / 2, ut = 4 * (ul >> 4);
  const bool v_mine = BITS == 4 && tid < Dp && ut < hi && ut + 4 > lo, v_part = v_mine && (lo > ut || hi < ut + 4);
  auto v_unit = [&](uint32_t kvh) __attribute__((always_inline)) {
    return (u32x2*)(sq.p.k + ((size_t)phys * KVH + kvh) * q4kv_block_bytes(Dp) + q4kv_v_bytes(Dp) + 8 * tid);
  };
  // The V word of two times four tokens' codes, a byte each: token r of the first in
  // nibble (r >> 1) + 4 (r & 1), of the second two nibbles on.
  auto v_word = [](uint32_t c0, uint32_t c1) __attribute__((always_inline)) {
    static_assert(q4kv_v_bit(1, 0) == 16 && q4kv_v_bit(2, 0) == 4 && q4kv_v_bit(3, 0) == 20 && q4kv_v_bit(0, 16) == 8, "V word");
    c0 &= 0x0F0F0F0Fu, c1 &= 0x0F0F0F0Fu;  // (a token that the call does not bring: whatever was there)
    return __builtin_amdgcn_perm(c1 | c1 >> 12, c0 | c0 >> 12, 0x05010400u);
  };
  uint32_t v_new = 0;  // nibbles of the call's tokens
#pragma unroll
  for (uint32_t r = 0; r < 4; ++r)
    if (ut + r >= lo && ut + r < hi) v_new |= 0x0F0Fu << q4kv_v_bit(r, 0);
  double *cos_d = (double*)table, *sin_d = cos_d + 16 * half;
  u32x2 old = {0u, 0u};
  if (v_part) old = *v_unit(kvh0);
  if (kTurns && half) {
    const uint32_t f = tid & ((1u << a.half_log) - 1);
    for (uint32_t slot = lo + (tid >> a.half_log); slot < hi && f < half; slot += threads >> a.half_log) {
      const uint32_t position = a.positions ? a.positions[base + slot] : 16 * page + slot;
      double sn, cs;
      sincos_f64((double)position * a.freq[f], &sn, &cs);
      cos_d[slot * half + f] = cs * a.factor;
      sin_d[slot * half + f] = sn * a.factor;
    }
    __syncthreads();
  }

  for (uint32_t kvh = kvh0; kvh < kvh1; ++kvh) {
    if (kTurns && half) {
      const double *cs = cos_d + there * half, *sn = sin_d + there * half;
      // (VEC: the four elements lie in the rotated part together, or not)
      if (!VEC || pair_of<INTERLEAVED>(d0, a.offset, a.rotary_dim).turned) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const Pair pr = pair_of<INTERLEAVED>(d0 + e, a.offset, a.rotary_dim);
          if (!VEC && !pr.turned) continue;
          const double y = pr.first ? -kp[e] : kp[e];
          x[0][e] = (float)(x[0][e] * cs[pr.freq] + y * sn[pr.freq]);
        }
      }
    }
    const size_t block = (size_t)phys * KVH + kvh;
    if constexpr (BITS == 4) {
      uint8_t* at = sq.p.k + block * q4kv_block_bytes(Dp);
      uint32_t word[2], u[2][4];
      q4kv_groups<VEC>(x, d0, D, word, u);
      // Two lanes hold a K word.
      uint32_t w = (u[0][0] | u[0][2] << 4 | u[0][1] << 16 | u[0][3] << 20) << (lane & 1 ? 8 : 0);
      static_assert(q4kv_k_bit(1) == 16 && q4kv_k_bit(2) == 4 && q4kv_k_bit(3) == 20 && q4kv_k_bit(4) == 8, "K word");
      w |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, 0xB1, 0xF, 0xF, false);
      if (mine) {
        if ((lane & 1) == 0) *(uint32_t*)(k_img + q4kv_k_word(Dp, slot, d0)) = w;
#pragma unroll
        for (int e = 0; e < 4; ++e) v_codes[(d0 + e) * kVRow + slot] = (uint8_t)u[1][e];
        if (i16 < 2) *(uint32_t*)(at + q4kv_scale_bytes(Dp) + 4 * q4kv_scale_word(Dp, i16, g, slot)) = i16 ? word[1] : word[0];
      }
    } else {
      int8_t kq[4], vq[4];
      const float ks = q8_rows_quant(x[0], G, kq), vs = q8_rows_quant(x[1], G, vq);
      if (mine) {
        *(uint32_t*)(sq.p.k + (block * 16 + slot) * Dp + d0) = pack_q8x4(kq);
#pragma unroll
        for (int e = 0; e < 4; ++e) v_codes[(d0 + e) * kVRow + slot] = (uint8_t)vq[e];
        if (i16 == 0 && g == 0) {
          sq.p.ks[block * 16 + slot] = ks;
          sq.p.vs[block * 16 + slot] = vs;
        }
      }
    }
    if (kvh + 1 < kvh1) load_head(kvh + 1);
    __syncthreads();

    if constexpr (BITS == 4) {
      if (tid < Dp) {
        if ((ul & 15) >= lo && (ul & 15) < hi)
          *(u32x2*)(sq.p.k + block * q4kv_block_bytes(Dp) + 8 * tid) = *(const u32x2*)(k_img + 8 * tid);
        if (v_mine) {
          const uint32_t d = 64 * (Dp == 64 ? 0 : 2 * (tid / 128) + tid % 2) + (ul & 15);
          u32x2 w;
#pragma unroll
          for (int j = 0; j < 2; ++j)
            w[j] = v_word(*(const uint32_t*)(v_codes + (d + 32 * j) * kVRow + ut),
                          *(const uint32_t*)(v_codes + (d + 32 * j + 16) * kVRow + ut));
          if (v_part) w = (w & v_new) | (old & ~v_new);
          *v_unit(kvh) = w;
          if (v_part && kvh + 1 < kvh1) old = *v_unit(kvh + 1);
        }
      }
    } else if (tid < Dp) {
      uint8_t* at = sq.p.v + (block * Dp + tid) * 16;
      if (lo == 0 && hi == 16) {
        *(u32x4*)at = *(const u32x4*)(v_codes + kVRow * tid);
      } else {
        for (uint32_t s = lo; s < hi; ++s) at[s] = v_codes[kVRow * tid + s];
      }
    }
    if (kvh + 1 < kvh1) __syncthreads();
  }
}

// Eight elements of a row from d on, as bf16.
template <bool VEC>
__device__ __forceinline__ void store8(uint16_t* row, uint32_t d, uint32_t dr, const float (&x)[8]) {
  if constexpr (VEC) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    *(u32x4*)(row + d) = w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (d + e < dr) row[d + e] = f32_to_bf16(x[e]);
  }
}

// Reads back (8192 tokens of 8 heads of 128: 12 us, 3.5 TB/s): a workgroup of 5/2 Dp
// threads a (page, KV head).  The first 2 Dp take 8
// elements of a key each, the others 8 dimensions of four tokens' values: the words
// (4 bits) or bytes (8) that hold them lie together for both.
template <int BITS, bool VEC>
__global__ __launch_bounds__(640) void kv_load_kernel(KvLoadArgs a) {
  const uint32_t KVH = a.kv_heads, D = a.head_dim, Dp = a.head_dim_pad;
  const uint32_t page = a.first / 16 + blockIdx.x / KVH, kvh = blockIdx.x % KVH;
  const size_t block = (size_t)a.p.pt[page] * KVH + kvh;
  const uint8_t* kv = a.p.k + block * q4kv_block_bytes(Dp);
  const uint32_t* scales = (const uint32_t*)(kv + q4kv_scale_bytes(Dp));
  const bool value = threadIdx.x >= 2 * Dp;
  const uint32_t i = threadIdx.x - (value ? 2 * Dp : 0), per = Dp / 8, d = i % per * 8;
  const uint32_t lo = max(a.first, 16 * page), hi = min(a.first + a.count, 16 * page + 16);  // tokens (no sum wraps)
  auto row = [&](uint16_t* out, uint32_t token) { return out + ((size_t)(token - a.first) * KVH + kvh) * D; };
  if (d >= D || !(value ? a.v : a.k)) return;
  float x[8];
  if (!value) {
    const uint32_t slot = i / per, token = 16 * page + slot;
    if (token < lo || token >= hi) return;
    if constexpr (BITS == 4) {
      const uint32_t w = scales[q4kv_scale_word(Dp, 0, d / 64, slot)], c = *(const uint32_t*)(kv + q4kv_k_word(Dp, slot, d));
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = q4kv_value((int)(c >> q4kv_k_bit(e) & 15) - 8, w);
    } else {
      const float s = a.p.ks[block * 16 + slot];
      const u32x2 c = *(const u32x2*)(a.p.k + (block * 16 + slot) * Dp + d);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)(int8_t)(c[e >> 2] >> (8 * (e & 3))) * s;
    }
    store8<VEC>(row(a.k, token), d, D, x);
    return;
  }
  const uint32_t slot0 = i / per * 4;
  uint32_t c[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    c[e] = BITS == 4 ? *(const uint32_t*)(kv + q4kv_v_bytes(Dp) + q4kv_v_word(Dp, slot0, d + e)) >> q4kv_v_bit(0, d)
                     : *(const uint32_t*)(a.p.v + (block * Dp + d + e) * 16 + slot0);
#pragma unroll
  for (uint32_t r = 0; r < 4; ++r) {
    const uint32_t token = 16 * page + slot0 + r;
    if (token < lo || token >= hi) continue;
    if constexpr (BITS == 4) {
      const uint32_t w = scales[q4kv_scale_word(Dp, 1, d / 64, slot0 + r)];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = q4kv_value((int)(c[e] >> q4kv_v_bit(r, 0) & 15) - 8, w);
    } else {
      const float s = a.p.vs[block * 16 + slot0 + r];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)(int8_t)(c[e] >> (8 * r)) * s;
    }
    store8<VEC>(row(a.v, token), d, D, x);
  }
}

template <int BITS, bool INTERLEAVED>
void launch_append(const KvAppendArgs& a, bool vec, bool qvec, uint32_t grid, hipStream_t st) {
  auto kernel = vec ? (qvec ? kv_append_kernel<BITS, uint16_t, INTERLEAVED, true, true>
                            : kv_append_kernel<BITS, uint16_t, INTERLEAVED, true, false>)
                    : (qvec ? kv_append_kernel<BITS, uint16_t, INTERLEAVED, false, true>
                            : kv_append_kernel<BITS, uint16_t, INTERLEAVED, false, false>);
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(4 * a.head_dim_pad), 16 * a.rotary_dim / 2 * 2 * sizeof(double), st, a);
}

// Gives every sequence its workgroups; returns how many there are.  A workgroup takes
// several KV heads of a page, which share its sines and cosines, where that leaves
// enough of them (16384 rows of 8 heads of 128: 116 us with one, 91 with up to eight).
uint64_t plan_units(KvAppendArgs* a) {
  constexpr uint64_t kEnough = 1024;
  auto pages = [](const KvAppendSeq& s) -> uint64_t {
    return s.rows ? (s.start + s.rows - 1) / 16 - s.start / 16 + 1 : 0;
  };
  uint64_t all = 0;
  for (uint32_t b = 0; b < a->n_seqs; ++b) all += pages(a->seqs[b]);
  a->share = 1;
  while (a->rotary_dim && a->share < 8 && a->share < a->kv_heads && all * ((a->kv_heads + 2 * a->share - 1) / (2 * a->share)) >= kEnough)
    a->share *= 2;
  a->half_log = 0;
  while (2u << a->half_log < a->rotary_dim) ++a->half_log;
  uint64_t units = 0;
  a->rows = 0;
  a->row0 = a->seqs[0].row0;
  for (uint32_t b = 0; b < a->n_seqs; ++b) {
    KvAppendSeq& s = a->seqs[b];
    s.unit_begin = (uint32_t)units;
    units += pages(s) * ((a->kv_heads + a->share - 1) / a->share);
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
    const uint32_t most = (a.q_items + 4 * a.head_dim_pad - 1) / (4 * a.head_dim_pad);
    a.q_groups = std::max(1u, std::min(most, (kQueryGroups + a.rows - 1) / a.rows));
    grid += (uint64_t)a.rows * a.q_groups;
  }
  if (grid > kv_append_most(a.head_dim_pad)) return hipErrorInvalidValue;
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
  if (grid > kv_append_most(a.head_dim_pad)) return hipErrorInvalidValue;
  auto kernel = vec ? kv_append_kernel<4, float, false, true, false> : kv_append_kernel<4, float, false, false, false>;
  hipLaunchKernelGGL(kernel, dim3((uint32_t)grid), dim3(4 * a.head_dim_pad), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_kv_load(const KvLoadArgs& a, uint32_t bits, hipStream_t st) {
  const uint64_t units = (uint64_t)((a.first + (uint64_t)a.count - 1) / 16 - a.first / 16 + 1) * a.kv_heads;
  if (a.count == 0 || units > kv_load_most(a.head_dim_pad)) return hipErrorInvalidValue;
  const bool vec = a.head_dim % 8 == 0 && (uintptr_t)a.k % 16 == 0 && (uintptr_t)a.v % 16 == 0;
  auto kernel = bits == 4 ? (vec ? kv_load_kernel<4, true> : kv_load_kernel<4, false>)
                          : (vec ? kv_load_kernel<8, true> : kv_load_kernel<8, false>);
  hipLaunchKernelGGL(kernel, dim3((uint32_t)units), dim3(5 * a.head_dim_pad / 2), 0, st, a);
  return hipGetLastError();
}

}  // namespace qm
