// GQA attention over the paged 4-bit KV cache (layout and codes: q4kv.h).
//
// A wave takes a (row, query head) and walks the row's tokens with a running
// maximum and sum; a lane holds the head's elements lane, lane + 64, ...
#include <float.h>

#include <type_traits>

#include "attention_device.h"
#include "kv_quant.h"
#include "q4kv.h"

namespace qm {
namespace {

// Exponent of values whose weights are kept low, so that sums of up to 2^22 of them stay finite.
constexpr int kBigValue = 96;

// One value of each DPP row for all 16 lanes of the row.
template <int I>
__device__ __forceinline__ float row_bcast(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + I, 0xF, 0xF, true));
}
template <int N, class F>
__device__ __forceinline__ void static_for(F f) {
  if constexpr (N > 0) {
    static_for<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

// Two words of signed nibbles (tokens 4 kq .. + 3 of d / 16 = 2 j, low half, and 2 j + 1)
// as bf16 of 16 c, exact.
__device__ __forceinline__ void v_operand(uint32_t w, u32x2& even, u32x2& odd) {
  const uint32_t hi = w & 0xF0F0F0F0u, lo = (w << 4) & 0xF0F0F0F0u;
  even = u32x2{pack_bf16x2((float)(int8_t)lo, (float)(int8_t)hi),
               pack_bf16x2((float)(int8_t)(lo >> 8), (float)(int8_t)(hi >> 8))};
  odd = u32x2{pack_bf16x2((float)(int8_t)(lo >> 16), (float)(int8_t)(hi >> 16)),
              pack_bf16x2((float)(int8_t)(lo >> 24), (float)(int8_t)(hi >> 24))};
}

// Eight bf16 of a query row from element d0 on, zero past the real dimension dr.
__device__ __forceinline__ u32x4 load_q8(const uint16_t* row, uint32_t d0, uint32_t dr) {
  if (dr % 8 == 0) return d0 < dr ? *(const u32x4*)(row + d0) : u32x4{0u, 0u, 0u, 0u};
  return load_bf16x8(row, d0, dr, false);
}

// What the words of a lane hold of one page (layout: q4kv.h).
template <int D>
struct PageRegs {
  static constexpr int kW = D / 32, kS = D == 256 ? 2 : 1;
  uint32_t k[kW], v[kW], s[kS];
};
template <int D>
__device__ __forceinline__ void load_part(__amdgpu_buffer_rsrc_t r, uint32_t base, int lane, uint32_t (&w)[D / 32]) {
  if constexpr (D == 64) {
    const auto x = __builtin_amdgcn_raw_buffer_load_b64(r, base + 8 * lane, 0, 0);
    w[0] = x[0], w[1] = x[1];
  } else {
#pragma unroll
    for (int j = 0; j < D / 128; ++j) {
      const auto x = __builtin_amdgcn_raw_buffer_load_b128(r, base + 1024 * j + 16 * lane, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[4 * j + i] = x[i];
    }
  }
}

template <int D, int W>
__global__ __launch_bounds__(64 * W, 2) void q4kv_decode_kernel(AttnArgs args) {
  constexpr int G = D / 64, kDB = D / 16, kRing = D == 256 ? 4 : 8;
  // Two waves a SIMD of D = 256 have no registers for the Q operand, which is the
  // same for all of them: it lies in LDS.
  constexpr bool kTight = D == 256;
  constexpr int kQBytes = kTight ? 2 * G * 1024 : 0;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kMergeBytes<D, W> + kQBytes];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kq = lane >> 4;
  const uint32_t H = args.heads, KVH = args.kv_heads, gh = H / KVH;

  uint32_t b = 0;
  const uint32_t unit = blockIdx.x;
  while (b + 1 < args.n_seqs && unit >= args.seqs[b + 1].unit_begin) ++b;
  const AttnSeq& sq = args.seqs[b];
  const uint32_t u = unit - sq.unit_begin;
  const uint32_t kvh = u % KVH, split = u / KVH;
  // Tokens read from pages: all but the one that this call brings.
  const bool append = args.k_new != nullptr;
  const uint32_t visible = sq.len - (append ? 1 : 0);
  const uint32_t pages = (visible + 15) / 16;
  const uint32_t p_begin = min(pages, split * args.pages_per_split);
  const uint32_t p_end = min(pages, p_begin + args.pages_per_split);
  const bool col_ok = (uint32_t)col < gh;
  const uint32_t head = kvh * gh + col;
  const uint32_t dr = args.head_dim;
  const float sm_scale = kLog2e / sqrtf((float)dr);

  // ---- this wave's pages: p_begin + wave + W j ------------------------------
  const uint32_t first = p_begin + wave;
  const uint32_t n_mine = first < p_end ? (p_end - first + W - 1) / W : 0;
  // Ids of the wave's next 64 pages (lane j: page j), taken with v_readlane; the 64
  // after them are on their way.
  auto load_ids = [&](uint32_t j0) __attribute__((always_inline)) {
    const uint32_t j = j0 + lane;
    return j < n_mine ? sq.pt[first + W * j] : 0;
  };
  int32_t ids = load_ids(0), ids_next = load_ids(64);
  const size_t block = (size_t)q4kv_block_bytes(D);
  // A page past the wave's last reads nothing: a buffer of no bytes.
  auto load = [&](uint32_t j) __attribute__((always_inline)) {
    if ((j & 63) == 0 && j > 0) {
      ids = ids_next;
      ids_next = load_ids(j + 64);
    }
    const int32_t phys = __builtin_amdgcn_readlane(ids, (int)(j & 63));
    const __amdgpu_buffer_rsrc_t r =
        make_rsrc((const uint8_t*)sq.k + ((size_t)phys * KVH + kvh) * block, j < n_mine ? (uint32_t)block : 0u);
    PageRegs<D> p;
    load_part<D>(r, 0, lane, p.k);
    if constexpr (D == 256) {
      p.s[0] = __builtin_amdgcn_raw_buffer_load_b32(r, q4kv_scale_bytes(D) + 4 * lane, 0, 0);
      p.s[1] = __builtin_amdgcn_raw_buffer_load_b32(r, q4kv_scale_bytes(D) + 256 + 4 * lane, 0, 0);
    } else {
      const uint32_t at = D == 128 ? lane : 8 * kq + (lane & 7);
      p.s[0] = __builtin_amdgcn_raw_buffer_load_b32(r, q4kv_scale_bytes(D) + 4 * at, 0, 0);
    }
    load_part<D>(r, q4kv_v_bytes(D), lane, p.v);
    return p;
  };

  // Q operand (B of K Q^T): the lane's 16 elements of every group, d = 64 g + 16 kq .. + 15.
  u32x4 qb[kTight ? 1 : 2 * G];
  u32x4* ql = (u32x4*)(lds + kMergeBytes<D, W>) + lane;
  {
    const uint16_t* qp = args.q + ((size_t)b * H + head) * dr;
    auto q_part = [&](int j) __attribute__((always_inline)) {
      return col_ok ? load_q8(qp, 64 * (j / 2) + 16 * kq + 8 * (j % 2), dr) : u32x4{0u, 0u, 0u, 0u};
    };
    if constexpr (kTight) {
      u32x4 x[2 * G / W];
#pragma unroll
      for (int j = 0; j < 2 * G / W; ++j) x[j] = q_part(wave + W * j);
#pragma unroll
      for (int j = 0; j < 2 * G / W; ++j) ql[64 * (wave + W * j)] = x[j];
    } else {
#pragma unroll
      for (int j = 0; j < 2 * G; ++j) qb[j] = q_part(j);
    }
  }
  auto q_of = [&](int j) __attribute__((always_inline)) { return kTight ? ql[64 * j] : qb[kTight ? 0 : j]; };
  PageRegs<D> ring[kRing];
#pragma unroll
  for (int r = 0; r < kRing; ++r) {
    ring[r] = load(r);
    // In order, or the loop's first wait would be for all of them.
    __builtin_amdgcn_sched_barrier(0);
  }
  if constexpr (kTight) lds_barrier();
  // Sums of the queries' groups, for the keys' offsets.
  float qs[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float x = 0.0f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const u32x4 q = q_of(2 * g + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) x += bf16_lo_f32(q[i]) + bf16_hi_f32(q[i]);
    }
    x += __shfl_xor(x, 16);
    qs[g] = x + __shfl_xor(x, 32);
  }

  floatx4 o[kDB];
#pragma unroll
  for (int i = 0; i < kDB; ++i) o[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  float om[G] = {};  // what the values' offsets add, a group each (this lane's tokens)
  float m_run = -INFINITY, l_lane = 0.0f;

  // ---- the token that this call brings ---------------------------------------
  // A wave with the fewest pages of the last split quantises it, writes it into its
  // page and starts its own softmax from it: no other wave waits, and nobody reads
  // the token back.  (Waves that read the page meanwhile see its other tokens'
  // nibbles in either version of a word, and give the new one no weight.)
  if (append && split + 1 == sq.nsplit && wave == (int)((p_end - p_begin) % W)) {
    const uint32_t token = sq.len - 1, slot = token % 16;
    const bool fresh = sq.new_page_count > 0;
    const int32_t phys = fresh ? sq.new_page_id : sq.pt[token / 16];
    if (fresh && kvh == 0 && lane == 0) sq.pt[token / 16] = phys;
    uint8_t* page = (uint8_t*)sq.k + ((size_t)phys * KVH + kvh) * block;
    float* xs = (float*)lds;               // values as the codes have them, K then V
    uint8_t* cs = lds + 2 * D * 4;         // codes, c & 15
    uint32_t old[D / 32];                  // the lane's V words of the page
#pragma unroll
    for (int w = 0; w < D / 32; ++w) old[w] = *(const uint32_t*)(page + q4kv_v_bytes(D) + q4kv_lane_word(D, lane, w));
    const uint32_t g = kq % G, d0 = 64 * g + 4 * col;
    float x[2][4];
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const float* src = (kind ? args.v_new : args.k_new) + ((size_t)b * KVH + kvh) * dr;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[kind][e] = d0 + e < dr ? src[d0 + e] : 0.0f;
    }
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      int c[4];
      const uint32_t w = q4kv_group(x[kind], d0, dr, c);
      if (kq >= G) continue;  // (copies of the first groups)
      floatx4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = q4kv_value(c[e], w);
      *(floatx4*)(xs + D * kind + d0) = y;
      *(uint32_t*)(cs + D * kind + d0) = (c[0] & 15) | (c[1] & 15) << 8 | (c[2] & 15) << 16 | (c[3] & 15) << 24;
      if (col == 0) *(uint32_t*)(page + q4kv_scale_bytes(D) + 4 * q4kv_scale_word(D, kind, g, slot)) = w;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if ((uint32_t)col == slot) {
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const uint8_t* c = cs + 64 * (j / 2) + 16 * kq + 8 * (j % 2);
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) w |= (uint32_t)(c[e] ^ 8) << q4kv_k_bit(e);
        *(uint32_t*)(page + q4kv_lane_word(D, lane, j)) = w;
      }
    }
    if ((uint32_t)kq == slot / 4) {
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const uint32_t sh = 4 * (slot % 4), c = cs[D + 32 * j + col] | cs[D + 32 * j + 16 + col] << 16;
        *(uint32_t*)(page + q4kv_v_bytes(D) + q4kv_lane_word(D, lane, j)) = (old[j] & ~(0x000F000Fu << sh)) | c << sh;
      }
    }
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < 2 * G; ++j) {
      const float* y = xs + 64 * (j / 2) + 16 * kq + 8 * (j % 2);
      const u32x4 q = q_of(j);
#pragma unroll
      for (int i = 0; i < 4; ++i) dot += bf16_lo_f32(q[i]) * y[2 * i] + bf16_hi_f32(q[i]) * y[2 * i + 1];
    }
    dot += __shfl_xor(dot, 16);
    dot += __shfl_xor(dot, 32);
    // Weight 1 against its own score, or less where the value is large (as below).
    float size = 0.0f;
#pragma unroll
    for (int i = 0; i < G; ++i) size = fmaxf(size, fabsf(xs[D + 64 * i + lane]));
    size = wave_allmax(size);
    const float excess = fmaxf(0.0f, (float)((int)(__float_as_uint(size) >> 23) - 127 - kBigValue));
    const float p = exp2f(-excess);
    m_run = dot * sm_scale + excess;
    l_lane = kq == 0 ? p : 0.0f;
#pragma unroll
    for (int db = 0; db < kDB; ++db) o[db] = *(const floatx4*)(xs + D + 16 * db + 4 * kq) * p;
    if (dot != dot) l_lane = dot;  // a NaN in the query or the key
  }

  const Q4KvUnpack k_operand;
  // Scores of two pages, S^T[token][col]: codes enter as 128 + (c + 8), exactly, and the
  // sums start 136 sums of the queries lower.
  auto qk = [&](const PageRegs<D>& pa, const PageRegs<D>& pb, float (&sc)[8]) __attribute__((always_inline)) {
    const float sa = bf16_lo_f32(pa.s[0]) * sm_scale, ma = bf16_hi_f32(pa.s[0]) * sm_scale;
    const float sb = bf16_lo_f32(pb.s[0]) * sm_scale, mb = bf16_hi_f32(pb.s[0]) * sm_scale;
    static_for<G>([&](auto gi) __attribute__((always_inline)) {
      constexpr int g = gi;
      const float c0 = -136.0f * qs[g];
      floatx4 a = {c0, c0, c0, c0}, c = a;
      const u32x4 q0 = q_of(2 * g), q1 = q_of(2 * g + 1);
      a = mfma16x16x32(k_operand(pa.k[2 * g]), q0, a);
      c = mfma16x16x32(k_operand(pb.k[2 * g]), q0, c);
      a = mfma16x16x32(k_operand(pa.k[2 * g + 1]), q1, a);
      c = mfma16x16x32(k_operand(pb.k[2 * g + 1]), q1, c);
      static_for<4>([&](auto ri) __attribute__((always_inline)) {
        constexpr int r = ri, i = 4 * g + r;
        const float xa = row_bcast<i>(ma) * qs[g], xb = row_bcast<i>(mb) * qs[g];
        sc[r] = __builtin_fmaf(row_bcast<i>(sa), a[r], g ? sc[r] + xa : xa);
        sc[4 + r] = __builtin_fmaf(row_bcast<i>(sb), c[r], g ? sc[4 + r] + xb : xb);
      });
      if constexpr (kTight) __builtin_amdgcn_sched_barrier(0);
    });
  };
  // Two pages a step: two independent score chains, one look at the running maximum,
  // then P'V with both pages' tokens in the K dimension.
  auto step = [&](PageRegs<D>& pa, PageRegs<D>& pb, uint32_t ja, auto may_be_last) __attribute__((always_inline)) {
    const bool last = decltype(may_be_last)::value && ja + 2 >= n_mine;
    constexpr int kVi = D == 256 ? 0 : 4 * G;  // the V items of a row's scale words
    const uint32_t ta = (first + W * ja) * 16 + 4 * kq, tb = ta + 16 * W;
    const bool has_b = ja + 1 < n_mine;
    if (last) {  // tokens past the last one have neither scale nor offset
#pragma unroll
      for (int i = 0; i < PageRegs<D>::kS; ++i) {
        if (ta + (lane & 3) >= visible) pa.s[i] = 0;
        if (!has_b || tb + (lane & 3) >= visible) pb.s[i] = 0;
      }
    }
    float sc[8];
    qk(pa, pb, sc);
    if (last) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (ta + r >= visible) sc[r] = -INFINITY;
        if (!has_b || tb + r >= visible) sc[4 + r] = -INFINITY;
      }
    }
    float bmax = sc[0];
#pragma unroll
    for (int r = 1; r < 8; ++r) bmax = fmaxf(bmax, sc[r]);
    bmax = max4_across_kq(bmax);
    // Values above 2^kBigValue weigh less from the start, so that their sums stay
    // finite: the reference covers score and size.
    const uint32_t wa = pa.s[PageRegs<D>::kS - 1], wb = pb.s[PageRegs<D>::kS - 1];
    {
      constexpr uint32_t kS = (127 + kBigValue - 4) << 7, kM = (127 + kBigValue) << 7;
      const bool big = (D == 256 || (lane & 15) >= kVi) && ((wa & 0x7F80u) >= kS || (wb & 0x7F80u) >= kS ||
                                                            (wa >> 16 & 0x7F80u) >= kM || (wb >> 16 & 0x7F80u) >= kM);
      if (__builtin_amdgcn_ballot_w64(big)) {
        const uint32_t e = max(max(wa >> 7 & 0xFF, wb >> 7 & 0xFF) + 4, max(wa >> 23 & 0xFF, wb >> 23 & 0xFF));
        bmax += wave_allmax(big ? (float)e - (127 + kBigValue) : 0.0f);
      }
    }
    // Lazy rescaling: the reference only moves when a score exceeds it by more than
    // 2^8 (see the 8-bit kernel).
    const float m_new = bmax > m_run + 8.0f ? bmax : m_run;
    const bool moved = m_new != m_run;
    if (__builtin_amdgcn_ballot_w64(moved)) {
      const float corr = moved ? exp2f(m_run - m_new) : 1.0f;
      l_lane *= corr;
#pragma unroll
      for (int db = 0; db < kDB; ++db) o[db] *= corr;
#pragma unroll
      for (int g = 0; g < G; ++g) om[g] *= corr;
    }
    m_run = m_new;
    float p[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      p[r] = __builtin_amdgcn_exp2f(sc[r] - m_new);
      l_lane += p[r];
    }
    // P' = p s / 16 as bf16 hi + lo (error 2^-17), a group each; V enters as signed
    // codes times 16: nothing accumulates into O but sum_t s c p.
    const float sa = bf16_lo_f32(wa) * 0.0625f, ma = bf16_hi_f32(wa);
    const float sb = bf16_lo_f32(wb) * 0.0625f, mb = bf16_hi_f32(wb);
    static_for<G>([&](auto gi) __attribute__((always_inline)) {
      constexpr int g = gi;
      float w[8];
      static_for<4>([&](auto ri) __attribute__((always_inline)) {
        constexpr int r = ri, i = kVi + 4 * g + r;
        w[r] = p[r] * row_bcast<i>(sa);
        w[4 + r] = p[4 + r] * row_bcast<i>(sb);
        om[g] += row_bcast<i>(ma) * p[r];
        om[g] += row_bcast<i>(mb) * p[4 + r];
      });
      u32x4 hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        hi[i] = pack_bf16x2(w[2 * i], w[2 * i + 1]);
        lo[i] = pack_bf16x2(w[2 * i] - bf16_lo_f32(hi[i]), w[2 * i + 1] - bf16_hi_f32(hi[i]));
      }
#pragma unroll
      for (int j = 2 * g; j < 2 * g + 2; ++j) {
        u32x2 ae, ao, be, bo;
        v_operand(pa.v[j], ae, ao);
        v_operand(pb.v[j], be, bo);
        const u32x4 even = {ae.x, ae.y, be.x, be.y}, odd = {ao.x, ao.y, bo.x, bo.y};
        o[2 * j] = mfma16x16x32(even, hi, o[2 * j]);
        o[2 * j + 1] = mfma16x16x32(odd, hi, o[2 * j + 1]);
        o[2 * j] = mfma16x16x32(even, lo, o[2 * j]);
        o[2 * j + 1] = mfma16x16x32(odd, lo, o[2 * j + 1]);
        if constexpr (kTight) __builtin_amdgcn_sched_barrier(0);
      }
    });
  };

  // Whole rounds of the ring, then what is left.  (A round that could end early would
  // make every wait in it one for nearly all loads.)
  uint32_t i = 0;
  for (; i + kRing < n_mine; i += kRing) {
#pragma unroll
    for (int s = 0; s < kRing; s += 2) {
      step(ring[s], ring[s + 1], i + s, BoolTag<false>{});
      ring[s] = load(i + s + kRing);
      ring[s + 1] = load(i + s + 1 + kRing);
    }
  }
#pragma unroll
  for (int s = 0; s < kRing; s += 2) {
    if (i + s >= n_mine) break;
    step(ring[s], ring[s + 1], i + s, BoolTag<true>{});
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float x = om[g] + __shfl_xor(om[g], 16);
    x += __shfl_xor(x, 32);
#pragma unroll
    for (int db = 4 * g; db < 4 * g + 4; ++db) o[db] += x;
  }
  decode_merge<D, W>(args, sq, b, kvh, split, lds, o, m_run, l_lane);
}

template <int D>
__global__ __launch_bounds__(64) void q4kv_attention_kernel(AttnArgs args) {
  constexpr int G = D / 64;
  const uint32_t H = args.heads, KVH = args.kv_heads, dr = args.head_dim;
  const uint32_t row = blockIdx.x / H, head = blockIdx.x % H, kvh = head / (H / KVH);
  const uint32_t lane = threadIdx.x;
  const AttnSeq& sq = args.seqs[args.prefill ? 0 : row];
  const uint32_t visible = args.prefill ? args.start + row + 1 : sq.len;
  const float scale = kLog2e / sqrtf((float)dr);
  float q[G], o[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const uint32_t d = 64 * g + lane;
    q[g] = d < dr ? bf16_to_f32(args.q[((size_t)row * H + head) * dr + d]) : 0.0f;
    o[g] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (uint32_t t = 0; t < visible; ++t) {
    const uint32_t slot = t % 16;
    const uint8_t* kv = (const uint8_t*)sq.k + ((size_t)sq.pt[t / 16] * KVH + kvh) * q4kv_block_bytes(D);
    const uint32_t* scales = (const uint32_t*)(kv + q4kv_scale_bytes(D));
    float dot = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint32_t d = 64 * g + lane;
      const int c = (int)(*(const uint32_t*)(kv + q4kv_k_word(D, slot, d)) >> q4kv_k_bit(d) & 15) - 8;
      if (d < dr) dot += q[g] * q4kv_value(c, scales[q4kv_scale_word(D, 0, g, slot)]);
    }
    const float s = wave_allsum(dot) * scale;
    // Values above 2^96 weigh less from the start, so that their sums stay finite:
    // the reference covers score and size.
    float size = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint32_t w = scales[q4kv_scale_word(D, 1, g, slot)];
      size = fmaxf(size, fmaxf(bf16_to_f32(w & 0xFFFFu), fabsf(__uint_as_float(w & 0xFFFF0000u))));
    }
    const float mn = fmaxf(m, s + fmaxf(0.0f, (float)((int)(__float_as_uint(size) >> 23) - 127 - kBigValue)));
    const float r = mn == -INFINITY ? 1.0f : exp2f(m - mn), p = exp2f(s - mn);
    l = l * r + p;
    m = mn;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint32_t d = 64 * g + lane;
      const int c = (int)((*(const uint32_t*)(kv + q4kv_v_bytes(D) + q4kv_v_word(D, slot, d)) >> q4kv_v_bit(slot, d) & 15) ^ 8) - 8;
      o[g] = o[g] * r + p * q4kv_value(c, scales[q4kv_scale_word(D, 1, g, slot)]);
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const uint32_t d = 64 * g + lane;
    if (d >= dr) continue;
    const size_t at = ((size_t)row * H + head) * dr + d;
    float v = o[g] / l;
    if (args.gate) v *= sigmoid_f(bf16_to_f32(args.gate[at]));
    args.o[at] = f32_to_bf16(v);
  }
}

template <int D>
hipError_t launch_d(const AttnArgs& a, uint32_t units, bool need_combine, hipStream_t st) {
  if (a.prefill) {
    hipLaunchKernelGGL(q4kv_attention_kernel<D>, dim3(a.rows * a.heads), dim3(64), 0, st, a);
    return hipGetLastError();
  }
  if (need_combine && !a.partials) return hipErrorInvalidValue;
  if (a.wg_waves == 8)
    hipLaunchKernelGGL((q4kv_decode_kernel<D, 8>), dim3(units), dim3(512), 0, st, a);
  else
    hipLaunchKernelGGL((q4kv_decode_kernel<D, 4>), dim3(units), dim3(256), 0, st, a);
  if (need_combine) launch_attn_combine(a, st);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_q4kv_attention(const AttnArgs& a, uint32_t units, bool need_combine, hipStream_t st) {
  switch (a.head_dim_pad) {
    case 64: return launch_d<64>(a, units, need_combine, st);
    case 128: return launch_d<128>(a, units, need_combine, st);
    case 256: return launch_d<256>(a, units, need_combine, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace qm
