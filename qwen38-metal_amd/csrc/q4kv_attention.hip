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
constexpr float kBigSize = 0x1p92f;  // of a scale or offset that may hold one

template <int N, class F>
__device__ __forceinline__ void static_for(F f) {
  if constexpr (N > 0) {
    static_for<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

// Products with one lane's value of every quad, x[r] (op)= (lane r's value) * y[r]: the
// broadcast rides on the multiplication as a DPP operand.  (The compiler folds it
// into plain products only; a multiply-add would get a copy.)  Each block begins
// with the two wait states that a DPP read needs after a VALU write.
#define QM_QUAD(op, x, v, y, r) op " %" #x ", %" #v ", %" #y " quad_perm:[" #r "," #r "," #r "," #r "] row_mask:0xf bank_mask:0xf\n"
// x[r] = v_r * y
__device__ __forceinline__ void quad_mul(float (&x)[4], float v, float y) {
  asm("s_nop 1\n" QM_QUAD("v_mul_f32_dpp", 0, 4, 5, 0) QM_QUAD("v_mul_f32_dpp", 1, 4, 5, 1)
      QM_QUAD("v_mul_f32_dpp", 2, 4, 5, 2) QM_QUAD("v_mul_f32_dpp", 3, 4, 5, 3)
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]) : "v"(v), "v"(y));
}
// x[r] += v_r * y
__device__ __forceinline__ void quad_fma(float (&x)[4], float v, float y) {
  asm("s_nop 1\n" QM_QUAD("v_fmac_f32_dpp", 0, 4, 5, 0) QM_QUAD("v_fmac_f32_dpp", 1, 4, 5, 1)
      QM_QUAD("v_fmac_f32_dpp", 2, 4, 5, 2) QM_QUAD("v_fmac_f32_dpp", 3, 4, 5, 3)
      : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]) : "v"(v), "v"(y));
}
// x[r] = v_r * y[r], sum += u_r * y[r]
__device__ __forceinline__ void quad_mul_sum(float (&x)[4], float& sum, float v, float u, const float (&y)[4]) {
  asm("s_nop 1\n" QM_QUAD("v_mul_f32_dpp", 0, 5, 7, 0) QM_QUAD("v_fmac_f32_dpp", 4, 6, 7, 0)
      QM_QUAD("v_mul_f32_dpp", 1, 5, 8, 1) QM_QUAD("v_fmac_f32_dpp", 4, 6, 8, 1)
      QM_QUAD("v_mul_f32_dpp", 2, 5, 9, 2) QM_QUAD("v_fmac_f32_dpp", 4, 6, 9, 2)
      QM_QUAD("v_mul_f32_dpp", 3, 5, 10, 3) QM_QUAD("v_fmac_f32_dpp", 4, 6, 10, 3)
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "+v"(sum)
      : "v"(v), "v"(u), "v"(y[0]), "v"(y[1]), "v"(y[2]), "v"(y[3]));
}
#undef QM_QUAD
template <int R>
__device__ __forceinline__ float quad_bcast(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), R * 0x55, 0xF, 0xF, true));
}

// Eight bf16 of a query row from element d0 on, zero past the real dimension dr.
__device__ __forceinline__ u32x4 load_q8(const uint16_t* row, uint32_t d0, uint32_t dr) {
  if (dr % 8 == 0) return d0 < dr ? *(const u32x4*)(row + d0) : u32x4{0u, 0u, 0u, 0u};
  return load_bf16x8(row, d0, dr, false);
}

// A lane's words of a pair of pages: codes of both, and the scale words (K's groups,
// then V's) of one token of one of them.
template <int D>
struct PairRegs {
  uint32_t k[2][D / 32], v[2][D / 32], s[D / 32];
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

// Decode: a workgroup takes up to 8 query heads of one KV head and a split of the
// pages.  Every wave walks its pages two at a time, straight from memory into
// registers, and the 16 columns of a matrix operand are 8 heads times the two pages:
//   S^T[token][column] = K Q^T with queries of zero in the other page's columns, so both
//   pages' products add up in one accumulator, each in its columns;
//   a lane's four scores are tokens 4 kq .. + 3 of its column's page, and its quad holds
//   these tokens' scale words, a lane each;
//   O^T[d][column] += V^T P'^T with both pages' tokens along K and P' of zero for
//   the other page.
// A column's softmax is its page's alone; decode_merge joins the columns of a head.
template <int D, int W>
__global__ __launch_bounds__(64 * W, 2) void q4kv_decode_kernel(AttnArgs args) {
  constexpr int G = D / 64, kDB = D / 16, kRing = D == 256 ? 2 : 4;  // pairs of pages in flight
  // Two waves a SIMD of D = 256 have no registers for the Q operands, which are the
  // same for all of them: they lie in LDS.
  constexpr bool kTight = D == 256;
  constexpr int kQBytes = kTight ? 4 * G * 1024 : 0;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kMergeBytes<D, W> + kQBytes];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kq = lane >> 4;
  const bool in_b = col >= 8;
  const uint32_t mask_b = in_b ? ~0u : 0u, mask_a = ~mask_b;
  const uint32_t H = args.heads, KVH = args.kv_heads, gh = H / KVH;

  uint32_t b = 0;
  const uint32_t unit = blockIdx.x;
  while (b + 1 < args.n_seqs && unit >= args.seqs[b + 1].unit_begin) ++b;
  const AttnSeq& sq = args.seqs[b];
  const uint32_t u = unit - sq.unit_begin, sets = q4kv_head_sets(gh);
  const uint32_t kvh = u % KVH, set = u / KVH % sets, split = u / (KVH * sets);
  const uint32_t per_set = (gh + sets - 1) / sets;
  const uint32_t head0 = kvh * gh + set * per_set, n_heads = min(per_set, gh - set * per_set);
  // Tokens read from pages: all but the one that this call brings.
  const bool append = args.k_new != nullptr;
  const uint32_t visible = sq.len - (append ? 1 : 0);
  const uint32_t pages = (visible + 15) / 16;
  const uint32_t p_begin = min(pages, split * args.pages_per_split);
  const uint32_t p_end = min(pages, p_begin + args.pages_per_split);
  const uint32_t head = head0 + (col & 7);
  const bool col_ok = (uint32_t)(col & 7) < n_heads;
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
  constexpr size_t block = q4kv_block_bytes(D);
  const uint32_t s_at = q4kv_scale_bytes(D) + 4 * q4kv_scale_word(D, 0, 0, 4 * kq + (lane & 3));
  // Pages j (even) and j + 1.  Codes of a page past the wave's last read nothing: a
  // buffer of no bytes.
  auto load = [&](uint32_t j) __attribute__((always_inline)) {
    if ((j & 63) == 0 && j > 0) {
      ids = ids_next;
      ids_next = load_ids(j + 64);
    }
    PairRegs<D> p;
    const uint8_t* page[2];
    __amdgpu_buffer_rsrc_t r[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int32_t phys = __builtin_amdgcn_readlane(ids, (int)((j + h) & 63));
      page[h] = (const uint8_t*)sq.k + ((size_t)phys * KVH + kvh) * block;
      r[h] = make_rsrc(page[h], j + h < n_mine ? (uint32_t)block : 0u);
      load_part<D>(r[h], 0, lane, p.k[h]);
    }
    // (A page id past the last is 0, whose memory is there.)
    const uint8_t* sp = (in_b ? page[1] : page[0]) + s_at;
    if constexpr (D == 64) {
      const u32x2 x = *(const u32x2*)sp;
      p.s[0] = x.x, p.s[1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < D / 128; ++i) {
        const u32x4 x = *(const u32x4*)(sp + 16 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) p.s[4 * i + e] = x[e];
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) load_part<D>(r[h], q4kv_v_bytes(D), lane, p.v[h]);
    return p;
  };

  // Q operands (B of K Q^T) of both pages: the lane's 16 elements of every group, d = 64 g
  // + 16 kq .. + 15.
  u32x4 qb[2][kTight ? 1 : 2 * G];
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
      for (int j = 0; j < 2 * G / W; ++j) {
        ql[64 * (wave + W * j)] = x[j] & mask_a;
        ql[64 * (2 * G + wave + W * j)] = x[j] & mask_b;
      }
    } else {
      u32x4 x[2 * G];
#pragma unroll
      for (int j = 0; j < 2 * G; ++j) x[j] = q_part(j);
#pragma unroll
      for (int j = 0; j < 2 * G; ++j) qb[0][j] = x[j] & mask_a, qb[1][j] = x[j] & mask_b;
    }
  }
  auto q_of = [&](int h, int j) __attribute__((always_inline)) {
    return kTight ? ql[64 * (2 * G * h + j)] : qb[h][kTight ? 0 : j];
  };
  PairRegs<D> ring[kRing];
#pragma unroll
  for (int r = 0; r < kRing; ++r) {
    ring[r] = load(2 * r);
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
      const u32x4 q = q_of(0, 2 * g + j) | q_of(1, 2 * g + j);
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
  floatx4 ow[G];     // -136 sums of P' since they last went into o (four times the same)
#pragma unroll
  for (int g = 0; g < G; ++g) ow[g] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_lane = 0.0f;

  // ---- the token that this call brings ---------------------------------------
  // A wave with the fewest pages of the last split quantises it, writes it into its
  // page (for the first heads' workgroup) and starts its own softmax from it: no
  // other wave waits, and nobody reads the token back.  (Waves that read the page
  // meanwhile see its other tokens' nibbles in either version of a word, and give
  // the new one no weight.)
  if (append && split + 1 == sq.nsplit && wave == (int)((p_end - p_begin) % W)) {
    const uint32_t token = sq.len - 1, slot = token % 16;
    const bool fresh = sq.new_page_count > 0;
    const int32_t phys = fresh ? sq.new_page_id : sq.pt[token / 16];
    uint8_t* page = (uint8_t*)sq.k + ((size_t)phys * KVH + kvh) * block;
    float* xs = (float*)lds;               // values as the codes have them, K then V
    uint8_t* cs = lds + 2 * D * 4;         // codes, c + 8
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
    uint32_t word[2];
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      int c[4];
      word[kind] = q4kv_group(x[kind], d0, dr, c);
      if (kq >= G) continue;  // (copies of the first groups)
      floatx4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = q4kv_value(c[e], word[kind]);
      *(floatx4*)(xs + D * kind + d0) = y;
      *(uint32_t*)(cs + D * kind + d0) = (c[0] + 8) | (c[1] + 8) << 8 | (c[2] + 8) << 16 | (c[3] + 8) << 24;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (set == 0) {
      if (fresh && kvh == 0 && lane == 0) sq.pt[token / 16] = phys;
      if (col == 0 && kq < G) {
#pragma unroll
        for (int kind = 0; kind < 2; ++kind)
          *(uint32_t*)(page + q4kv_scale_bytes(D) + 4 * q4kv_scale_word(D, kind, g, slot)) = word[kind];
      }
      if ((uint32_t)col == slot) {
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const uint8_t* c = cs + 64 * (j / 2) + 16 * kq + 8 * (j % 2);
          uint32_t w = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) w |= (uint32_t)c[e] << q4kv_k_bit(e);
          *(uint32_t*)(page + q4kv_lane_word(D, lane, j)) = w;
        }
      }
      if ((uint32_t)kq == slot / 4) {
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const uint32_t sh = q4kv_v_bit(slot, 0), c = cs[D + 32 * j + col] | cs[D + 32 * j + 16 + col] << 8;
          *(uint32_t*)(page + q4kv_v_bytes(D) + q4kv_lane_word(D, lane, j)) = (old[j] & ~(0x0F0Fu << sh)) | c << sh;
        }
      }
    }
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < 2 * G; ++j) {
      const float* y = xs + 64 * (j / 2) + 16 * kq + 8 * (j % 2);
      const u32x4 q = q_of(0, j);
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
    const float p = in_b ? 0.0f : exp2f(-excess);
    if (!in_b) m_run = dot * sm_scale + excess;
    l_lane = kq == 0 ? p : 0.0f;
    if (!in_b) {
#pragma unroll
      for (int db = 0; db < kDB; ++db) o[db] = *(const floatx4*)(xs + D + 16 * db + 4 * kq) * p;
    }
    if (dot != dot) l_lane = dot;  // a NaN in the query or the key
  }

  const Q4KvUnpack unpack;
  const u32x4 minus136 = {0xC308C308u, 0xC308C308u, 0xC308C308u, 0xC308C308u};
  auto step = [&](PairRegs<D>& pg, uint32_t j, auto may_be_last) __attribute__((always_inline)) {
    const bool last = decltype(may_be_last)::value && j + 2 >= n_mine;
    // This lane's page: its first token of four, and the end of what it may see.
    const uint32_t t0 = (first + W * (j + (in_b ? 1 : 0))) * 16 + 4 * kq;
    const uint32_t end = in_b && j + 1 >= n_mine ? 0 : visible;
    if (last && t0 + (lane & 3) >= end) {  // tokens past the last one have neither scale nor offset
#pragma unroll
      for (int i = 0; i < D / 32; ++i) pg.s[i] = 0;
    }
    // Scores: codes enter as 128 + (c + 8), exactly, and the sums start 136 sums of the
    // queries lower.
    float x[4];
    static_for<G>([&](auto gi) __attribute__((always_inline)) {
      constexpr int g = gi;
      const float c0 = -136.0f * qs[g];
      floatx4 acc = {c0, c0, c0, c0};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 2 * g; i < 2 * g + 2; ++i) acc = mfma16x16x32(unpack(pg.k[h][i]), q_of(h, i), acc);
      const float sk = bf16_lo_f32(pg.s[g]) * sm_scale, mk = bf16_hi_f32(pg.s[g]) * sm_scale;
      if (g == 0) quad_mul(x, mk, qs[g]);
      else quad_fma(x, mk, qs[g]);
      static_for<4>([&](auto ri) __attribute__((always_inline)) {
        constexpr int r = ri;
        x[r] = __builtin_fmaf(quad_bcast<r>(sk), acc[r], x[r]);
      });
      if constexpr (kTight) __builtin_amdgcn_sched_barrier(0);
    });
    if (last) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (t0 + r >= end) x[r] = -INFINITY;
    }
    float bmax = max4_across_kq(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    // Values above 2^kBigValue weigh less from the start, so that their sums stay
    // finite: the reference covers score and size.
    float size = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g)
      size = fmaxf(size, fmaxf(bf16_lo_f32(pg.s[G + g]), fabsf(bf16_hi_f32(pg.s[G + g]))));
    if (__builtin_amdgcn_ballot_w64(size > kBigSize))
      bmax += fmaxf(0.0f, wave_allmax((float)(int)(__float_as_uint(size) >> 23)) + (4 - 127 - kBigValue));
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
      for (int g = 0; g < G; ++g) om[g] *= corr, ow[g] *= corr;
    }
    m_run = m_new;
    float p[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      p[r] = __builtin_amdgcn_exp2f(x[r] - m_new);
      // (a column that has seen nothing: its reference is -inf too)
      if (decltype(may_be_last)::value && x[r] == -INFINITY) p[r] = 0.0f;
      l_lane += p[r];
    }
    // P' = p s as bf16 hi + lo (error 2^-17), a group each.  Values enter as 128 + (c + 8)
    // too; the sum of 136 P' that they bring along is formed by the same operands
    // against -136, so its roundings of P' are the same, and goes into O every round.
    static_for<G>([&](auto gi) __attribute__((always_inline)) {
      constexpr int g = gi;
      float w[4];
      quad_mul_sum(w, om[g], bf16_lo_f32(pg.s[G + g]), bf16_hi_f32(pg.s[G + g]), p);
      const uint32_t h01 = pack_bf16x2(w[0], w[1]), h23 = pack_bf16x2(w[2], w[3]);
      const uint32_t l01 = pack_bf16x2(w[0] - bf16_lo_f32(h01), w[1] - bf16_hi_f32(h01));
      const uint32_t l23 = pack_bf16x2(w[2] - bf16_lo_f32(h23), w[3] - bf16_hi_f32(h23));
      const u32x4 hi = {h01 & mask_a, h23 & mask_a, h01 & mask_b, h23 & mask_b};
      const u32x4 lo = {l01 & mask_a, l23 & mask_a, l01 & mask_b, l23 & mask_b};
      ow[g] = mfma16x16x32(minus136, hi, ow[g]);
      ow[g] = mfma16x16x32(minus136, lo, ow[g]);
#pragma unroll
      for (int i = 2 * g; i < 2 * g + 2; ++i) {
        const u32x4 va = unpack(pg.v[0][i]), vb = unpack(pg.v[1][i]);
        const u32x4 even = {va.x, va.y, vb.x, vb.y}, odd = {va.z, va.w, vb.z, vb.w};
        o[2 * i] = mfma16x16x32(even, hi, o[2 * i]);
        o[2 * i + 1] = mfma16x16x32(odd, hi, o[2 * i + 1]);
        o[2 * i] = mfma16x16x32(even, lo, o[2 * i]);
        o[2 * i + 1] = mfma16x16x32(odd, lo, o[2 * i + 1]);
        if constexpr (kTight) __builtin_amdgcn_sched_barrier(0);
      }
    });
  };
  auto settle = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int db = 4 * g; db < 4 * g + 4; ++db) o[db] += ow[g];
      ow[g] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
  };

  // Whole rounds of the ring, then what is left.  (A round that could end early would
  // make every wait in it one for nearly all loads.)
  uint32_t i = 0;
  for (; i + 2 * kRing < n_mine; i += 2 * kRing) {
#pragma unroll
    for (int s = 0; s < kRing; ++s) {
      step(ring[s], i + 2 * s, BoolTag<false>{});
      ring[s] = load(i + 2 * s + 2 * kRing);
    }
    settle();
  }
#pragma unroll
  for (int s = 0; s < kRing; ++s) {
    if (i + 2 * s >= n_mine) break;
    step(ring[s], i + 2 * s, BoolTag<true>{});
  }
  settle();
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float x = om[g] + __shfl_xor(om[g], 16);
    x += __shfl_xor(x, 32);
#pragma unroll
    for (int db = 4 * g; db < 4 * g + 4; ++db) o[db] += x;
  }
  decode_merge<D, W, 2>(args, sq, b, head0, n_heads, split, lds, o, m_run, l_lane);
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
      const int c = (int)(*(const uint32_t*)(kv + q4kv_v_bytes(D) + q4kv_v_word(D, slot, d)) >> q4kv_v_bit(slot, d) & 15) - 8;
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
