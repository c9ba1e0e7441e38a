// GQA attention over the paged 4-bit KV cache (layout and codes: q4kv.h).
//
// With x = s c + m for every element of a group g, what attention needs splits into
// products of codes, which matrix instructions form exactly, and a few products a token:
//   q . k = sum_g s_g (q_g . c_g) + m_g (sum of q_g),
//   sum_t p_t v_t = sum_t (p_t s_t) c_t + (sum_t p_t m_t)      (decode).
// Decode reads every page once, straight into registers, and is bound by that stream and
// by its vector instructions; prefill unpacks a tile once for up to 256 columns and is
// bound by the issue of its vector and matrix instructions.  Softmax with a running
// reference and sum in fp32.
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

// Ends a decode workgroup.  Lane (col, kq) of a wave holds o[db][r] for d = 16 db + 4 kq
// + r of column col, its reference m and its own share of the sum of weights l.  Head
// head0 + c has columns c and c + 8 of every wave: all meet in LDS, in 16-byte pieces
// (rows of D + 4 floats spread 16 columns over the banks), and every thread weighs
// them by itself.  They leave as outputs, or as one split's partials.
constexpr int kMergeRow(int D) { return D + 4; }
template <int D, int W>
constexpr int kMergeBytes = W * 16 * (kMergeRow(D) * 4 + 8);
template <int D, int W>
__device__ __forceinline__ void merge_columns(const AttnCommon& args, const Q4KvSeq& sq, uint32_t b, uint32_t head0,
                                              uint32_t n_heads, uint32_t split, uint8_t* lds,
                                              const floatx4 (&o)[D / 16], float m, float l_lane) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kq = lane >> 4;
  const uint32_t H = args.heads, dr = args.head_dim;
  const float l = sum4_across_kq(l_lane);
  float* sums = (float*)lds;                               // [wave][column][kMergeRow(D)]
  float4* ml = (float4*)(sums + W * 16 * kMergeRow(D));  // [head][wave]: m, l of both columns
#pragma unroll
  for (int db = 0; db < D / 16; ++db)
    *(floatx4*)(sums + (16 * wave + col) * kMergeRow(D) + 16 * db + 4 * kq) = o[db];
  if (kq == 0) ((float2*)ml)[((col & 7) * W + wave) * 2 + (col >> 3)] = float2{m, l};
  lds_barrier();
  for (uint32_t e = threadIdx.x; e < n_heads * (D / 4); e += 64 * W) {
    const uint32_t c = e / (D / 4), d0 = 4 * (e % (D / 4)), head = head0 + c;
    float4 x[W];
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      x[w] = ml[c * W + w];
      mx = fmaxf(mx, fmaxf(x[w].x, x[w].z));
    }
    floatx4 O = {0.f, 0.f, 0.f, 0.f};
    float L = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // (a column that saw nothing holds zeros)
        const float mw = h ? x[w].z : x[w].x, f = mw == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw - mx);
        O += *(const floatx4*)(sums + (16 * w + 8 * h + c) * kMergeRow(D) + d0) * f;
        L += (h ? x[w].w : x[w].y) * f;
      }
    if (sq.nsplit > 1) {
      // Partials: O [split row][H][D], then (m, l) [split row][H][2].
      const size_t row = (size_t)(sq.part_begin + split) * H + head;
      *(floatx4*)(args.partials + row * D + d0) = O;
      if (d0 == 0) *(float2*)(args.partials + (size_t)args.part_rows * H * D + row * 2) = float2{mx, L};
      continue;
    }
    if (d0 >= dr) continue;
    O *= 1.0f / fmaxf(L, FLT_MIN);
    const size_t at = ((size_t)b * H + head) * dr + d0;
    if (args.out8) {
      *(u32x2*)(args.o + at) = args.gate ? gated_bf16x4(O, *(const u32x2*)(args.gate + at)) : bf16x4_of(O);
    } else {
      for (int i = 0; i < 4 && d0 + i < dr; ++i) {
        float v = O[i];
        if (args.gate) v *= gate_sigmoid(bf16_to_f32(args.gate[at + i]));
        args.o[at + i] = f32_to_bf16(v);
      }
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
// A column's softmax is its page's alone; merge_columns joins the columns of a head.
//
// Weights P' = p s are bf16 hi + lo (error 2^-17), codes exact.  131072 tokens of 24 / 4
// heads of 256: 36.7 us, 151 MB at 4.1 TB/s (a copy reaches 4.7), vector instructions
// busy for 40 % of the cycles, matrix ones for 14 %; 16 sequences of 32768 tokens of 64 / 8
// heads of 128: 117 us, 604 MB at 5.2 TB/s (the loads alone 109).  With one page a round,
// its 8 heads in 8 of the 16 columns, a ragged batch of 8 took 71.8 us against 66.1.
template <int D, int W>
__global__ __launch_bounds__(64 * W, D == 256 && W == 4 ? 1 : 2) void q4kv_decode_kernel(Q4KvArgs args) {
  constexpr int G = D / 64, kDB = D / 16, kRing = D == 256 ? 2 : 4;  // pairs of pages in flight
  // Two waves a SIMD of D = 256 have no registers for the Q operands, which are the
  // same for all of them: they lie in LDS, and the columns' sums of their 8-element
  // pieces behind them.
  constexpr bool kTight = D == 256 && W == 8;
  constexpr int kQBytes = kTight ? 4 * G * 1024 + 16 * 2 * G * 4 : 0;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kMergeBytes<D, W> + kQBytes];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kq = lane >> 4;
  const bool in_b = col >= 8;
  const uint32_t mask_b = in_b ? ~0u : 0u, mask_a = ~mask_b;
  const uint32_t H = args.heads, KVH = args.kv_heads, gh = H / KVH;

  // Its sequence: a lane looks at each (one load, where a search would wait for several).
  const uint32_t unit = blockIdx.x;
  uint32_t b = 0;
  if (args.n_seqs > 1)
    b = __builtin_popcountll(__builtin_amdgcn_ballot_w64((uint32_t)lane < args.n_seqs && unit >= args.seqs[lane].unit_begin)) - 1;
  const Q4KvSeq& sq = args.seqs[b];
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
  constexpr size_t block = q4kv_block_bytes(D);
  // The wave that takes the token that this call brings (below) has its loads under way
  // first.
  const bool takes_new = append && split + 1 == sq.nsplit && wave == (int)((p_end - p_begin) % W);
  const bool fresh = sq.new_page_count > 0;
  int32_t new_phys = sq.new_page_id;
  float xn[2][4];  // elements 4 col .. + 3 of group kq % G, of the key and of the value
  if (takes_new) {
    if (!fresh) new_phys = sq.pt[(sq.len - 1) / 16];
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const float* src = (kind ? args.v_new : args.k_new) + ((size_t)b * KVH + kvh) * dr;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t d = 64 * (kq % G) + 4 * col + e;
        xn[kind][e] = d < dr ? src[d] : 0.0f;
      }
    }
  }
  int32_t ids = load_ids(0), ids_next = load_ids(64);
  // The lane's pieces of the queries, 8 elements: piece j holds d = 64 (j / 2) + 16 kq + 8
  // (j % 2) .. + 7.
  constexpr int kMine = kTight ? 2 * G / W : 2 * G;
  u32x4 qx[kMine];
  auto piece_of = [&](int i) { return kTight ? wave + W * i : i; };
  if (dr % 8 == 0) {
    // One buffer for the sequence's queries: what is not there reads as zero, with no
    // branch whose end would wait for the loads.
    const __amdgpu_buffer_rsrc_t r = make_rsrc(args.q + (size_t)b * H * dr, H * dr * 2);
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const uint32_t d0 = 64 * (piece_of(i) / 2) + 16 * kq + 8 * (piece_of(i) % 2);
      const auto x = __builtin_amdgcn_raw_buffer_load_b128(r, col_ok && d0 < dr ? 2 * (head * dr + d0) : ~0u, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) qx[i][e] = x[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kMine; ++i)
      qx[i] = col_ok ? load_q8(args.q + ((size_t)b * H + head) * dr, 64 * (piece_of(i) / 2) + 16 * kq + 8 * (piece_of(i) % 2), dr)
                     : u32x4{0u, 0u, 0u, 0u};
  }
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
      page[h] = sq.k + ((size_t)phys * KVH + kvh) * block;
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

  PairRegs<D> ring[kRing];
#pragma unroll
  for (int r = 0; r < kRing; ++r) {
    ring[r] = load(2 * r);
    // In order, or the loop's first wait would be for all of them.
    __builtin_amdgcn_sched_barrier(0);
  }
  // The word that the new token shares with others of its page, in every piece.
  uint8_t* const new_page = sq.k + ((size_t)new_phys * KVH + kvh) * block;
  uint32_t old[D / 32];
  if (takes_new) {
#pragma unroll
    for (int w = 0; w < D / 32; ++w)
      old[w] = *(const uint32_t*)(new_page + q4kv_v_bytes(D) + q4kv_lane_word(D, lane, w));
  }
  // Q operands (B of K Q^T) of both pages, and the sums of the queries' groups for the
  // keys' offsets.
  u32x4 qb[2][kTight ? 1 : 2 * G];
  u32x4* ql = (u32x4*)(lds + kMergeBytes<D, W>) + lane;
  float qs[G];
  {
    float piece[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      float x = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) x += bf16_lo_f32(qx[i][e]) + bf16_hi_f32(qx[i][e]);
      piece[i] = x;
    }
    if constexpr (kTight) {
      float* sums = (float*)(lds + kMergeBytes<D, W> + 4 * G * 1024);  // [column][piece]
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int j = wave + W * i;
        ql[64 * j] = qx[i] & mask_a;
        ql[64 * (2 * G + j)] = qx[i] & mask_b;
        piece[i] = sum4_across_kq(piece[i]);
        if (kq == 0) sums[2 * G * col + j] = piece[i];
      }
      lds_barrier();
#pragma unroll
      for (int g = 0; g < G; ++g) qs[g] = sums[2 * G * col + 2 * g] + sums[2 * G * col + 2 * g + 1];
    } else {
#pragma unroll
      for (int j = 0; j < 2 * G; ++j) qb[0][j] = qx[j] & mask_a, qb[1][j] = qx[j] & mask_b;
#pragma unroll
      for (int g = 0; g < G; ++g) qs[g] = sum4_across_kq(piece[kTight ? 0 : 2 * g] + piece[kTight ? 0 : 2 * g + 1]);
    }
  }
  auto q_of = [&](int h, int j) __attribute__((always_inline)) {
    return kTight ? ql[64 * (2 * G * h + j)] : qb[h][kTight ? 0 : j];
  };

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
  if (takes_new) {
    const uint32_t token = sq.len - 1, slot = token % 16;
    // In the wave's own part of LDS (others may be about to leave their sums in theirs).
    float* xs = (float*)lds + 16 * wave * kMergeRow(D);  // values as the codes have them, K then V
    uint8_t* cs = (uint8_t*)(xs + 2 * D);                  // codes, c + 8
    const uint32_t g = kq % G, d0 = 64 * g + 4 * col;
    uint32_t word[2], u[2][4];
    q4kv_groups<false>(xn, d0, dr, word, u);
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      if (kq >= G) continue;  // (copies of the first groups)
      floatx4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = q4kv_value((int)u[kind][e] - 8, word[kind]);
      *(floatx4*)(xs + D * kind + d0) = y;
      *(uint32_t*)(cs + D * kind + d0) = u[kind][0] | u[kind][1] << 8 | u[kind][2] << 16 | u[kind][3] << 24;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (set == 0) {
      if (fresh && kvh == 0 && lane == 0) sq.pt[token / 16] = new_phys;
      if (col == 0 && kq < G) {
#pragma unroll
        for (int kind = 0; kind < 2; ++kind)
          *(uint32_t*)(new_page + q4kv_scale_bytes(D) + 4 * q4kv_scale_word(D, kind, g, slot)) = word[kind];
      }
      if ((uint32_t)col == slot) {
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const uint8_t* c = cs + 64 * (j / 2) + 16 * kq + 8 * (j % 2);
          uint32_t w = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) w |= (uint32_t)c[e] << q4kv_k_bit(e);
          *(uint32_t*)(new_page + q4kv_lane_word(D, lane, j)) = w;
        }
      }
      if ((uint32_t)kq == slot / 4) {
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const uint32_t sh = q4kv_v_bit(slot, 0), c = cs[D + 32 * j + col] | cs[D + 32 * j + 16 + col] << 8;
          *(uint32_t*)(new_page + q4kv_v_bytes(D) + q4kv_lane_word(D, lane, j)) = (old[j] & ~(0x0F0Fu << sh)) | c << sh;
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
    dot = sum4_across_kq(dot);
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
    const float x = sum4_across_kq(om[g]);
#pragma unroll
    for (int db = 4 * g; db < 4 * g + 4; ++db) o[db] += x;
  }
  merge_columns<D, W>(args, sq, b, head0, n_heads, split, lds, o, m_run, l_lane);
}

// Causal prefill on 32x32x16 MFMA; columns and tiles as in the 8-bit kernel, splits too
// or by block (Q4KvPrefillArgs).  A tile's 32 tokens are unpacked once per workgroup:
//   K as its codes in bf16 (16 c, exact), so a group's product is exact and its scale
//     and offset act on the scores: x = sum_g s_g (K_g Q_g) + m_g (sum of Q_g).  The
//     second part and the running reference come from one more matrix instruction,
//     whose K dimension holds m_g against three bf16 terms of the sums, and ones
//     against three of minus the reference.
//   V as values in fp16 in units of 2^R, where the largest of the first tile are 2^6 .. 2^7.
//     The weight of P V is p in fp16 with a reference that keeps it between 2^-24 and
//     2^15.5: one product instead of the two of a split P' (V and p round by 2^-11 at most
//     each), and what is lost is weights below 2^-36 of the row's largest.
//   That holds while the sizes of all tokens' groups (8 s or |m|: no value passes twice that)
//     lie between 2^-8 and 2^14 of the unit: above, fp16 ends; below, its steps of 2^-24 begin
//     to count.  A workgroup that meets another size starts again (prefill_far).
// The tables of a tile (scales, offsets, powers) are formed a tile ahead of its
// unpacking by two waves.
//
// 2048 rows on 4096 tokens of 64 / 8 heads of 128: 472 us, 727 TFLOP/s (a large matrix
// product reaches 1230), matrix instructions busy for 30 % of the cycles, vector ones
// for 42 %, half of those for the unpacking and the softmax's exponentials.  Before the
// values had one unit (457 us) the same took 618 without scores a tile ahead, and 564 with a
// tile's tables and V on the last waves alone.  1000 rows of 24 / 4 heads of 256, the kernel
// alone: 50 us (about 70 with the same number of workgroups for every block of columns).
constexpr uint32_t kHasNan = 1, kHasWide = 2;
// Sizes below it (values of the least scale) count as none.
constexpr float kNoSize = 0x1p-121f;
template <int D, int W>
struct PrefillLds {
  static constexpr int G = D / 64;
  // Two waves a SIMD of D = 256: half of the Q operand waits in LDS, and a tile's scores
  // are formed, a group at a time, in the step that uses them.
  static constexpr bool kTight = D == 256 && W == 8;
  // One barrier a tile: K of a tile and the next, V of the last one too.
  static constexpr int kNK = 2, kNV = kTight ? 2 : 3, kNTabs = 3;
  static constexpr int kK = 32 * D * 2, kV = 32 * D * 2;
  // A tile's tables: K scales [G][32], K offsets as matrix operand [2][32] of 16 bytes,
  // V scales and offsets in fp16 [G][8 token quads] of 16 bytes, then 2^R, what the tile has
  // of kHas.., and a word per group: tokens whose values are NaN.
  static constexpr int kKb = G * 128, kVs = kKb + 1024, kMisc = kVs + G * 128, kNan = kMisc + 16, kTab = kMisc + 32;
  static constexpr int kVAt = kNK * kK, kTabs = kVAt + kNV * kV;
  static constexpr int kIds = kTabs + kNTabs * kTab;
  static constexpr int kQ = kIds + 512, kQSteps = kTight ? D / 32 : 0;
  static constexpr int kBytes = kQ + W * kQSteps * 1024;
};

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float2_t __attribute__((ext_vector_type(2)));
// (By value: a bit cast of a vector's element takes its first.)
__device__ __forceinline__ half2_t as_half2(uint32_t x) { return __builtin_bit_cast(half2_t, x); }
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2_t){a, b}, half2_t));
}
__device__ __forceinline__ floatx16 mfma32x32x16_f16(u32x4 a, u32x4 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0,
                                                0, 0);
}
// The eight codes of a V word in fp16: 0x6400 | u is the fp16 1024 + u, of which 1032
// leaves c, exactly.
struct Q4KvUnpackF16 {
  uint32_t mask = 0x000F000Fu, one = 0x64006400u;
  __device__ __forceinline__ Q4KvUnpackF16() { asm("" : "+s"(mask), "+v"(one)); }
  __device__ __forceinline__ void operator()(uint32_t w, half2_t (&c)[4]) const {
    const half2_t bias = {(_Float16)-1032.0f, (_Float16)-1032.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = as_half2((w >> (4 * i) & mask) | one) + bias;
  }
};
// x as three bf16 terms, 24 bits together.
__device__ __forceinline__ void split3(float x, uint32_t (&t)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    t[i] = pack_bf16x2(x, 0.0f);
    x -= bf16_lo_f32(t[i]);
  }
}
// Eight codes of a K word as bf16 of 16 c, in order.
__device__ __forceinline__ u32x4 k_codes16(uint32_t w) {
  w ^= 0x88888888u;  // c in two's complement
  const uint32_t hi = w & 0xF0F0F0F0u, lo = (w << 4) & 0xF0F0F0F0u;
  auto f = [](uint32_t x, int b) { return (float)(int8_t)(x >> (8 * b)); };
  // Nibbles of elements 0 .. 7: 0, 4, 1, 5, 2, 6, 3, 7.
  return u32x4{pack_bf16x2(f(lo, 0), f(lo, 2)), pack_bf16x2(f(hi, 0), f(hi, 2)), pack_bf16x2(f(lo, 1), f(lo, 3)),
               pack_bf16x2(f(hi, 1), f(hi, 3))};
}

// What a wave of the prompts' kernel does: tiles t0 .. t1 - 1 for columns c0 .. c0 + 31, of
// which a lane has column c, a query head of a row.
struct PrefillPlace {
  uint32_t kvh, split, splits, t0, t1, c0, cols, c, row, head, visible;
  bool col_ok;
};
template <int W>
__device__ __forceinline__ PrefillPlace prefill_place(const Q4KvPrefillArgs& args, uint32_t workgroup, uint32_t wave,
                                                      uint32_t lane) {
  const uint32_t lc = lane & 31;
  const uint32_t KVH = args.kv_heads, gh = args.heads / KVH, len = args.seqs[0].len;  // gh <= 16
  PrefillPlace p;
  // Workgroups as in the 8-bit kernel: a KV head's on the same XCDs, the longest first.
  p.cols = args.rows * gh;
  const uint32_t blocks = (p.cols + 32 * W - 1) / (32 * W);
  const uint32_t bs = workgroup / KVH;
  uint32_t split = bs % args.splits, rb = blocks - 1 - bs / args.splits;
  if (args.split_tiles) {
    uint32_t first = 0;
    split = 0;
#pragma unroll
    for (int s = 1; s < kMaxBlockSplits; ++s)
      if (bs >= args.split_begin[s]) split = s, first = args.split_begin[s];
    rb = blocks - 1 - (bs - first);
  }
  p.kvh = workgroup % KVH;
  p.split = __builtin_amdgcn_readfirstlane(split);
  rb = __builtin_amdgcn_readfirstlane(rb);
  p.c0 = rb * 32 * W + wave * 32;
  // Columns past the last one repeat it and are not stored.
  p.c = min(p.c0 + lc, p.cols - 1);
  p.col_ok = p.c0 + lc < p.cols;
  p.row = p.c / gh, p.head = p.kvh * gh + (p.c - p.row * gh);
  p.visible = min(args.start + p.row + 1, len);
  const uint32_t tiles = prefill_tiles(rb, 32 * W, p.cols, gh, args.start, len);
  p.splits = prefill_block_splits(tiles, args.split_tiles, args.splits);
  p.t0 = (uint32_t)((uint64_t)tiles * p.split / p.splits), p.t1 = (uint32_t)((uint64_t)tiles * (p.split + 1) / p.splits);
  return p;
}
// Whether a block leaves partials.  One split needs none; with gates, blocks that have
// workgroups of their own leave them all the same, as the merge applies those with the
// whole chip.
__device__ __forceinline__ bool leaves_partials(const Q4KvPrefillArgs& args, const PrefillPlace& p) {
  return p.splits > 1 || (args.split_tiles && args.gate);
}

// A wave's columns where sizes are far apart, a group of 64 dimensions at a time: no LDS,
// few registers, K, V and Q straight from memory (2048 rows on 4096 tokens of 64 / 8
// heads of 128: 4.6 ms against 0.46; 333 rows of 20 / 5 heads of 80: 65 us against 18).  The
// other form's loop with groups and bands of its own was faster here, but the compiler then
// spilled in both (0.51 to 0.71 ms for ordinary values).  The values of a token are in units of their own power of two, 2^e, O
// in those of the group's largest so far, 2^R, and the weights are p 2^(e - R), taken to the
// products in bands of 2^24 with a power of two for every column that makes a band's
// largest 2^11 .. 2^12.  Nothing but parts below 2^-96 of the group's largest value is lost.
template <int D, int W>
__device__ __forceinline__ void prefill_far(const Q4KvPrefillArgs& args, uint32_t wave) {
  constexpr int G = D / 64;
  // (Formed anew: what both forms need would be held in registers over the other's loop.)
  uint32_t workgroup = blockIdx.x, none = 0;
  asm volatile("" : "+s"(workgroup), "+s"(wave), "+s"(none));
  int lane = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, none));
  const PrefillPlace p = prefill_place<W>(args, workgroup, wave, lane);
  if (p.c0 >= p.cols) return;
  int lc = lane & 31, hf = lane >> 5;
  const AttnSeq& sq = args.seqs[0];
  const uint32_t H = args.heads, KVH = args.kv_heads, dr = args.head_dim, last_page = (sq.len - 1) / 16;
  const float sm_scale = kLog2e / sqrtf((float)dr);
  const uint16_t* qp = args.q + ((size_t)p.row * H + p.head) * dr;
  auto token_of = [&](int e) __attribute__((always_inline)) { return 8 * (e >> 2) + 4 * hf + (e & 3); };
  auto power = [](float size) { return max((int)(__float_as_uint(size) >> 23) - 140, -113); };  // (up to 114)
#pragma unroll 1
  for (uint32_t g = 0; g < G; ++g) {
    floatx16 o[2] = {floatx16{}, floatx16{}};
    float m_run = 0.0f, l_lane = 0.0f;
    int r_exp = -113;
#pragma unroll 1
    for (uint32_t t = p.t0; t < p.t1; ++t) {
      asm volatile("" : "+v"(lane));
      lc = lane & 31, hf = lane >> 5;
      const uint8_t* block[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        block[h] = (const uint8_t*)sq.k + ((size_t)sq.pt[min(2 * t + h, last_page)] * KVH + p.kvh) * q4kv_block_bytes(D);
      const uint8_t* own = lc & 16 ? block[1] : block[0];  // the page of token 32 t + lc
      const uint32_t* scales = (const uint32_t*)(own + q4kv_scale_bytes(D));
      const uint32_t slot = lc & 15;
      const bool there = 32 * t + lc < sq.len;
      floatx16 x{};
#pragma unroll 1
      for (uint32_t i = 0; i < G; ++i) {
        floatx16 sc{};
        float qs = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t d0 = 64 * i + 16 * j + 8 * hf;
          const u32x4 q = load_q8(qp, d0, dr);
#pragma unroll
          for (int e = 0; e < 4; ++e) qs += bf16_lo_f32(q[e]) + bf16_hi_f32(q[e]);
          sc = mfma32x32x16(k_codes16(*(const uint32_t*)(own + q4kv_k_word(D, slot, d0))), q, sc);
          __builtin_amdgcn_sched_barrier(0);
        }
        qs += __shfl_xor(qs, 32);
        const uint32_t w = there ? scales[q4kv_scale_word(D, 0, i, slot)] : 0;
        const float sk = bf16_lo_f32(w) * (sm_scale * 0.0625f), mk = bf16_hi_f32(w) * sm_scale;  // (codes are 16 c)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          x[e] = __builtin_fmaf(__shfl(sk, token_of(e)), sc[e], __builtin_fmaf(__shfl(mk, token_of(e)), qs, x[e]));
          if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
      }
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        if (32 * t + token_of(e) >= p.visible) x[e] = -INFINITY;
        top = fmaxf(top, x[e]);
      }
      top = max2_across_halves(top);
      if (top > -INFINITY && (t == p.t0 || top > m_run + 12.0f)) {
        const float corr = t == p.t0 ? 0.0f : __builtin_amdgcn_exp2f(m_run - top);
        m_run = top;
        l_lane *= corr;
        o[0] *= corr, o[1] *= corr;
      }
      // The values' sizes, as in the other form.
      const uint32_t w = there ? scales[q4kv_scale_word(D, 1, g, slot)] : 0;
      const float sv = bf16_lo_f32(w), mv = bf16_hi_f32(w), size = fmaxf(8.0f * sv, fabsf(mv));
      const bool any = size >= kNoSize, bad = sv != sv;
      const float row_top = row_allmax(any ? size : 0.0f);
      const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(row_top), __float_as_uint(row_top), false, false);
      const uint32_t most = __builtin_amdgcn_readfirstlane(max(sw[0], sw[1]));  // (not negative)
      if (most != 0 && power(__uint_as_float(most)) > r_exp + 1) {
        const float unit = __builtin_amdgcn_exp2f((float)(r_exp - power(__uint_as_float(most))));
        r_exp = power(__uint_as_float(most));
        o[0] *= unit, o[1] *= unit;
      }
      const int e_own = any ? power(size) : r_exp;
      const float inv = __uint_as_float((uint32_t)(127 - e_own) << 23);
      const uint32_t sm = bad ? 0u : pack_f16x2(sv * inv, mv * inv);
      const float part = any ? (float)(e_own - r_exp) : -INFINITY;  // (a token without a size takes no part)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        l_lane += __builtin_amdgcn_exp2f(x[e] - m_run);
        x[e] += __shfl(part, token_of(e)) - m_run;
        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
      // V^T operands: tokens 4 hf .. + 3 and 8 + 4 hf .. + 3 of either page.
      u32x4 v[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          half2_t s_m[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) s_m[r] = as_half2(__shfl(sm, 16 * h + 8 * n + 4 * hf + r));
#pragma unroll
          for (int db = 0; db < 2; ++db) {
            const uint32_t d = 64 * g + 32 * db + lc;
            const uint32_t codes = *(const uint32_t*)(block[h] + q4kv_v_bytes(D) + q4kv_v_word(D, 8 * n + 4 * hf, d));
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
              y[r] = __builtin_fmaf((float)((int)(codes >> q4kv_v_bit(r, d) & 15) - 8), (float)s_m[r][0], (float)s_m[r][1]);
            v[h][db][2 * n] = pack_f16x2(y[0], y[1]), v[h][db][2 * n + 1] = pack_f16x2(y[2], y[3]);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      float below = INFINITY;
      for (int pass = 0; pass < 6; ++pass) {  // (weights are 2^12 at most: six reach below 2^-110)
        float high = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (x[e] < below) high = fmaxf(high, x[e]);
        high = max2_across_halves(high);
        if (!__builtin_amdgcn_ballot_w64(high > -110.0f)) break;
        const float low = high - 24.0f, unit = fmaxf(ceilf(high - 12.0f), -122.0f), back = __builtin_amdgcn_exp2f(unit);
        floatx16 band[2] = {floatx16{}, floatx16{}};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            y[e] = x[8 * h + e] < below && x[8 * h + e] >= low ? __builtin_amdgcn_exp2f(x[8 * h + e] - unit) : 0.0f;
          const u32x4 b = {pack_f16x2(y[0], y[1]), pack_f16x2(y[2], y[3]), pack_f16x2(y[4], y[5]), pack_f16x2(y[6], y[7])};
          band[0] = mfma32x32x16_f16(v[h][0], b, band[0]);
          band[1] = mfma32x32x16_f16(v[h][1], b, band[1]);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e)
          o[0][e] = __builtin_fmaf(band[0][e], back, o[0][e]), o[1][e] = __builtin_fmaf(band[1][e], back, o[1][e]);
        below = low;
      }
      // Values that are NaN: of the columns that see them.  (A NaN in a weight is in l.)
      const uint32_t n = p.visible > 32 * t ? p.visible - 32 * t : 0, seen = n >= 32 ? ~0u : (1u << n) - 1;
      if ((uint32_t)__builtin_amdgcn_ballot_w64(bad) & seen) {
#pragma unroll
        for (int e = 0; e < 16; ++e) o[0][e] = o[1][e] = NAN;
      }
    }
    const float l_tot = l_lane + __shfl_xor(l_lane, 32);
    const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot, unit = __uint_as_float((uint32_t)(127 + r_exp) << 23);
    if (!p.col_ok) continue;
    const bool partials = leaves_partials(args, p);
    const size_t pr = ((size_t)p.row * args.splits + p.split) * H + p.head, at = ((size_t)p.row * H + p.head) * dr;
#pragma unroll
    for (int db = 0; db < 2; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t d = 64 * g + 32 * db + token_of(e);
        float y = o[db][e] * inv * unit;
        if (partials) {
          args.partials[pr * D + d] = y;
        } else if (d < dr) {
          if (args.gate) y *= gate_sigmoid(bf16_to_f32(args.gate[at + d]));
          args.o[at + d] = f32_to_bf16(y);
        }
      }
    if (partials && g == 0 && hf == 0)
      *(float2*)(args.partials + (size_t)args.part_rows * H * D + pr * 2) =
          l_tot == 0.0f ? float2{-FLT_MAX, 0.0f} : float2{m_run + log2f(l_tot), 1.0f};
  }
}

// A workgroup's tiles; false, and no output, where sizes are far apart.  (What is rare is
// marked so: the compiler gives registers to the loops that it takes for frequent, and
// those of prefill_far are nested.)
template <int D, int W>
__device__ __forceinline__ bool prefill_block(const Q4KvPrefillArgs& args, uint8_t* lds, const int wave) {
  using L = PrefillLds<D, W>;
  constexpr int G = D / 64;
  constexpr int kDB = D / 32;  // 32-wide d blocks of O^T
  constexpr int kKS = D / 16;  // QK k-steps
  constexpr int kWords = 4 * D >= 64 * W ? 4 * D / (64 * W) : 1;  // words of a tile's K, and of its V, per thread
  constexpr float kMost = 15.5f;  // exponents above it move the reference
  constexpr int kNoUnit = 127;    // R where no tile has had a size
  const int lane = threadIdx.x & 63;
  const int lc = lane & 31, hf = lane >> 5;
  const uint32_t H = args.heads, KVH = args.kv_heads, gh = H / KVH;
  const AttnSeq& sq = args.seqs[0];
  const PrefillPlace place = prefill_place<W>(args, blockIdx.x, wave, lane);
  const uint32_t kvh = place.kvh, t0 = place.t0, t1 = place.t1, c0 = place.c0, cols = place.cols;
  const uint32_t row = place.row, head = place.head, visible = place.visible;
  const uint32_t last_page = (sq.len - 1) / 16;

  const uint32_t dr = args.head_dim;
  const float sm_scale = kLog2e / sqrtf((float)dr);
  constexpr bool kTight = L::kTight;
  constexpr int kQReg = kKS - L::kQSteps;
  u32x4 qb[kQReg];
  u32x4* ql = (u32x4*)(lds + L::kQ + wave * L::kQSteps * 1024) + lane;
  // What the bias product multiplies: three terms of every group's sum of queries (half
  // 0 holds slots 0..7, half 1 slots 8..15), and of minus the reference in slots 12..14.
  u32x4 qbias;
  {
    const uint16_t* qp = args.q + ((size_t)row * H + head) * dr;
    float qs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kKS; ++s) {
      const u32x4 x = load_q8(qp, 16 * s + 8 * hf, dr);
#pragma unroll
      for (int i = 0; i < 4; ++i) qs[s / 4] += bf16_lo_f32(x[i]) + bf16_hi_f32(x[i]);
      if (s < kQReg) qb[s < kQReg ? s : 0] = x;
      else ql[64 * (s - kQReg)] = x;
    }
    uint32_t t[4][3];
#pragma unroll
    for (int g = 0; g < 4; ++g) split3((qs[g] + __shfl_xor(qs[g], 32)) * sm_scale, t[g]);
    qbias = hf == 0 ? u32x4{t[0][0] | t[0][1] << 16, t[0][2] | t[1][0] << 16, t[1][1] | t[1][2] << 16,
                            t[2][0] | t[2][1] << 16}
                    : u32x4{t[2][2] | t[3][0] << 16, t[3][1] | t[3][2] << 16, 0u, 0u};
  }

  floatx16 o[kDB];
#pragma unroll
  for (int i = 0; i < kDB; ++i) o[i] = floatx16{};
  float m_run = 0.0f, l_lane = 0.0f;  // (the first tile sets the reference)

  // Without registers to spare, what depends on the lane alone is formed anew each step.
  auto anew = [](int x) __attribute__((always_inline)) {
    if (kTight) asm volatile("" : "+v"(x));
    return x;
  };
  // A thread's words of a tile: kWords in a row of its 4 D words of K, and the same of V
  // (2 D a page; the page is uniform over a wave).
  struct Raw {
    uint32_t k[kWords], v[kWords];
  };
  struct Pages {
    u32x2 id;
  };
  constexpr bool kAll = 4 * D >= 64 * W;  // every wave has words
  const int page_half = wave * 64 * kWords / (2 * D);
  const uint32_t word0 = (wave * 64 + lane) * kWords % (2 * D);
  // Ids of the pages of 64 tiles wait in LDS, 32 tiles ahead.  (Held in registers over
  // the loop they would be copied at its end, with a wait for every load in flight.)
  auto load_ids = [&](uint32_t t) __attribute__((always_inline)) {  // of tiles t .. t + 31
    ((int32_t*)(lds + L::kIds))[2 * ((t - t0) & 63) + lane] = sq.pt[min(2 * t + lane, last_page)];
  };
  auto page_ids = [&](uint32_t t) __attribute__((always_inline)) {
    return Pages{*(const u32x2*)(lds + L::kIds + 8 * ((t - t0) & 63))};
  };
  auto block_of = [&](uint32_t phys) __attribute__((always_inline)) {
    return (const uint8_t*)sq.k + ((size_t)(int32_t)phys * KVH + kvh) * q4kv_block_bytes(D);
  };
  auto load_words = [&](const uint8_t* p, uint32_t (&w)[kWords]) __attribute__((always_inline)) {
    if constexpr (kWords == 1) {
      w[0] = *(const uint32_t*)p;
    } else if constexpr (kWords == 2) {
      const u32x2 x = *(const u32x2*)p;
      w[0] = x.x, w[1] = x.y;
    } else {
      const u32x4 x = *(const u32x4*)p;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = x[i];
    }
  };
  auto fetch = [&](const Pages& ph, Raw& r) __attribute__((always_inline)) {
    if (!kAll && wave >= 4 * D / 64) return;
    const uint8_t* p = block_of(__builtin_amdgcn_readfirstlane(page_half ? ph.id.y : ph.id.x)) + 4 * word0;
    load_words(p, r.k);
    load_words(p + q4kv_v_bytes(D), r.v);
  };
  // Scale words of K (wave 0) and V (wave 1): a token a lane, twice.
  struct Words {
    uint32_t w[G];
  };
  auto fetch_words = [&](const Pages& ph, Words& r) __attribute__((always_inline)) {
    if (wave >= 2) return;
    const uint8_t* p = block_of(lc & 16 ? ph.id.y : ph.id.x) + q4kv_scale_bytes(D) + 4 * q4kv_scale_word(D, wave, 0, lc & 15);
    if constexpr (G == 1) {
      r.w[0] = *(const uint32_t*)p;
    } else if constexpr (G == 2) {
      const u32x2 x = *(const u32x2*)p;
      r.w[0] = x.x, r.w[1] = x.y;
    } else {
      const u32x4 x = *(const u32x4*)p;
#pragma unroll
      for (int g = 0; g < 4; ++g) r.w[g] = x[g];
    }
  };
  auto table = [&](uint32_t t) __attribute__((always_inline)) { return lds + L::kTabs + t % L::kNTabs * L::kTab; };
  int r_exp = kNoUnit;  // R (wave 1's)
  auto write_table = [&](uint32_t t, Words r) __attribute__((always_inline)) {
    if (wave >= 2) return;
    uint8_t* tab = table(t);
    if (32 * t + lc >= sq.len) {  // slots past the last token hold whatever was there
#pragma unroll
      for (int g = 0; g < G; ++g) r.w[g] = 0;
    }
    if (wave == 0) {
      uint32_t m[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int g = 0; g < G; ++g) {
        *(float*)(tab + 128 * g + 4 * lc) = bf16_lo_f32(r.w[g]) * (sm_scale * 0.0625f);  // (codes are 16 c)
        m[g] = r.w[g] >> 16;
      }
      *(u32x4*)(tab + L::kKb + 16 * lc) =
          u32x4{m[0] | m[0] << 16, m[0] | m[1] << 16, m[1] | m[1] << 16, m[2] | m[2] << 16};
      // Slots 12..14: ones for the reference.
      *(u32x4*)(tab + L::kKb + 512 + 16 * lc) = u32x4{m[2] | m[3] << 16, m[3] | m[3] << 16, 0x3F803F80u, 0x3F80u};
      return;
    }
    // Sizes of the tokens' values, NaN aside.
    float most = 0.0f, least = INFINITY;
    bool nan = false;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float sv = bf16_lo_f32(r.w[g]), size = fmaxf(8.0f * sv, fabsf(bf16_hi_f32(r.w[g])));
      most = fmaxf(most, size);
      least = fminf(least, size >= kNoSize ? size : INFINITY);
      nan |= sv != sv;
    }
    if (r_exp == kNoUnit) {
      const float x = row_allmax(most);
      const auto sw = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
      const uint32_t top = __builtin_amdgcn_readfirstlane(max(sw[0], sw[1]));
      if (__uint_as_float(top) >= kNoSize) r_exp = max((int)(top >> 23) - (127 + 6), -126);
    }
    // (Before there is a unit, values of the least scale alone: zeros.)
    const int e = r_exp == kNoUnit ? 0 : r_exp;
    const float unit = __uint_as_float((uint32_t)(127 + e) << 23), inv = __uint_as_float((uint32_t)(127 - e) << 23);
    uint32_t has = __builtin_amdgcn_ballot_w64(most >= unit * 0x1p14f || least < unit * 0x1p-8f) ? kHasWide : 0;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float sv = bf16_lo_f32(r.w[g]);
      const bool bad = sv != sv;
      _Float16* at = (_Float16*)(tab + L::kVs + 16 * (8 * g + (lc >> 2)) + 2 * (lc & 3));
      at[0] = (_Float16)(bad ? 0.0f : sv * inv);
      at[4] = (_Float16)(bad ? 0.0f : bf16_hi_f32(r.w[g]) * inv);
    }
    if (__builtin_amdgcn_ballot_w64(nan)) {
      has |= kHasNan;
#pragma unroll
      for (int g = 0; g < G; ++g)
        *(uint32_t*)(tab + L::kNan + 4 * g) = (uint32_t)__builtin_amdgcn_ballot_w64((r.w[g] & 0x7FFFu) > 0x7F80u);
    }
    *(float2*)(tab + L::kMisc) = float2{unit, __uint_as_float(has)};
  };
  // LDS images: K 16-byte chunk (8 d) q of token t at unit 32 q + (t ^ swz), V^T chunk
  // (page, half, d) at unit (2 page + half) D + (d ^ swz), where half 0 holds a page's
  // tokens 0..3, 8..11 and half 1 tokens 4..7, 12..15.  The swizzles spread what
  // neighbouring threads write over the banks.
  auto k_unit = [](uint32_t q, uint32_t tok) { return 32 * q + (tok ^ ((q >> 1 & 7) ^ (q & 1) << 1)); };
  auto v_unit = [](uint32_t half, uint32_t d) { return half * D + (d ^ (d >> 3 & 12)); };
  auto k_tile = [&](uint32_t t) __attribute__((always_inline)) { return lds + t % L::kNK * L::kK; };
  auto v_tile = [&](uint32_t t) __attribute__((always_inline)) { return lds + L::kVAt + t % L::kNV * L::kV; };
  const Q4KvUnpackF16 unpack;
  auto stage_in = [&](uint32_t t, const Raw& r) __attribute__((always_inline)) {
    if (!kAll && wave >= 4 * D / 64) return;
    uint8_t *kl = k_tile(t), *vl = v_tile(t);
    const uint8_t* tab = table(t);
#pragma unroll
    for (int n = 0; n < kWords; ++n) {
      const uint32_t wi = (wave * 64 + anew(lane)) * kWords % (2 * D) + n;
      const uint32_t l = D == 64 ? wi / 2 : wi % 256 / 4, j = D == 64 ? wi % 2 : 4 * (wi / 256) + wi % 4;
      const uint32_t low = l & 15, kq = l >> 4;
      // d = 64 (j / 2) + 16 kq + 8 (j % 2) .. + 7
      *(u32x4*)(kl + 16 * k_unit(8 * (j / 2) + 2 * kq + j % 2, 16 * page_half + low)) = k_codes16(r.k[n]);
      const u32x4 sm = *(const u32x4*)(tab + L::kVs + 16 * (8 * (j / 2) + 4 * page_half + kq));
      const half2_t s01 = as_half2(sm.x), s23 = as_half2(sm.y), m01 = as_half2(sm.z), m23 = as_half2(sm.w);
      half2_t c[4];  // tokens 0, 1 and 2, 3 of d / 16 = 2 j, then of 2 j + 1
      unpack(r.v[n], c);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const half2_t a = __builtin_elementwise_fma(c[2 * i], s01, m01), b = __builtin_elementwise_fma(c[2 * i + 1], s23, m23);
        *(u32x2*)(vl + 16 * v_unit(2 * page_half + (kq & 1), 32 * j + 16 * i + low) + 8 * (kq >> 1)) =
            u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
      }
    }
  };

  u32x4 ph[2];  // the weights of a tile, two k-steps
  floatx16 x, sc[kTight ? 1 : G];
  auto scaled = [&](uint32_t t, const floatx16& s, int g) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const floatx4 k = ((const floatx4*)(table(t) + 128 * g))[2 * i + hf];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * i + e] = __builtin_fmaf(s[4 * i + e], k[e], x[4 * i + e]);
    }
  };
  // Scores of tile t: their offsets and reference in x, the groups' products in sc.
  auto products = [&](uint32_t t) __attribute__((always_inline)) {
    const int lc = anew(lane) & 31, hf = anew(lane) >> 5;
    const u32x4* kl = (const u32x4*)k_tile(t);
    x = mfma32x32x16(*(const u32x4*)(table(t) + L::kKb + 16 * lane), qbias, floatx16{});
    if constexpr (kTight) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        sc[0] = floatx16{};
#pragma unroll
        for (int j = 4 * g; j < 4 * g + 4; ++j) {
          sc[0] = mfma32x32x16(kl[k_unit(2 * j + hf, lc)], j < kQReg ? qb[j < kQReg ? j : 0] : ql[64 * (j - kQReg)], sc[0]);
          __builtin_amdgcn_sched_barrier(0);
        }
        scaled(t, sc[0], g);
      }
    } else {
#pragma unroll
      for (int g = 0; g < G; ++g) sc[g] = floatx16{};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const int j = 4 * g + i;
          sc[g] = mfma32x32x16(kl[k_unit(2 * j + hf, lc)], qb[j], sc[g]);
        }
    }
  };
  auto add_values = [&](uint32_t t) __attribute__((always_inline)) {
    const int lc = anew(lane) & 31, hf = anew(lane) >> 5;
    const u32x4* vl = (const u32x4*)v_tile(t);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int db = 0; db < kDB; ++db) {
        o[db] = mfma32x32x16_f16(vl[v_unit(2 * j + hf, 32 * db + lc)], ph[j], o[db]);
        if (kTight) __builtin_amdgcn_sched_barrier(0);
      }
  };

  // Weights of tile t.  MASKED is false for tiles every column of the wave sees whole.
  bool near = true;
  auto weights = [&](uint32_t t, auto masked) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked)::value;
    const uint8_t* tab = table(t);
    // (the same in every lane)
    const uint32_t has = __builtin_amdgcn_readfirstlane(*(const uint32_t*)(tab + L::kMisc + 4));
    if (__builtin_expect_with_probability((has & kHasWide) != 0, false, 1.0)) near = false;
    if constexpr (!kTight) {
#pragma unroll
      for (int g = 0; g < G; ++g) scaled(t, sc[g], g);
    }
    // Element e is token 32 t + 8 (e >> 2) + 4 hf + (e & 3).
    float xmax = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if (MASKED && 32 * t + 8 * (e >> 2) + 4 * hf + (e & 3) >= visible) x[e] = -INFINITY;
      xmax = fmaxf(xmax, x[e]);
    }
    if (__builtin_expect(t == t0 || __builtin_amdgcn_ballot_w64(xmax > kMost), 0)) {
      xmax = max2_across_halves(xmax);
      // Whole numbers: the largest weight becomes 2^11 .. 2^12.
      const float shift = (t == t0 || xmax > kMost) && xmax > -INFINITY ? ceilf(xmax - 12.0f) : 0.0f;
      m_run += shift;
      const float corr = __builtin_amdgcn_exp2f(-shift);
      if (t != t0) {  // (nothing is there yet in the first tile, and corr may be infinite)
        l_lane *= corr;
#pragma unroll
        for (int db = 0; db < kDB; ++db) o[db] *= corr;
      }
      uint32_t r[3];
      split3(-m_run, r);
      if (hf) qbias.z = r[0] | r[1] << 16, qbias.w = r[2];
      x -= shift;
    }
    // The sum takes the weights before they round.
    float psum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float w0 = __builtin_amdgcn_exp2f(x[2 * i]), w1 = __builtin_amdgcn_exp2f(x[2 * i + 1]);
      ph[i >> 2][i & 3] = pack_f16x2(w0, w1);
      psum[0] += w0, psum[1] += w1;
    }
    l_lane += psum[0] + psum[1];
    if (__builtin_expect(has & kHasNan, 0)) {  // values that are NaN: of the columns that see them, and their group
      const uint32_t n = visible > 32 * t ? visible - 32 * t : 0, seen = n >= 32 ? ~0u : (1u << n) - 1;
#pragma unroll
      for (int g = 0; g < G; ++g)
        if (*(const uint32_t*)(tab + L::kNan + 4 * g) & seen) {
#pragma unroll
          for (int db = 2 * g; db < 2 * g + 2; ++db)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[db][e] = NAN;
        }
    }
  };

  Raw raw{};
  Words words{};
  if (t0 < t1) {
    if (wave == 0) load_ids(t0);
    lds_barrier();
    Words w0{}, w1{};
    Raw r0{};
    const Pages p0 = page_ids(t0), p1 = page_ids(t0 + 1), p2 = page_ids(t0 + 2);
    fetch_words(p0, w0);
    fetch_words(p1, w1);
    fetch(p0, r0);
    fetch(p1, raw);
    fetch_words(p2, words);
    write_table(t0, w0);
    write_table(t0 + 1, w1);
    lds_barrier();
    stage_in(t0, r0);
  }
  lds_barrier();
  // A wave without columns only unpacks (not for D = 128, where the branch keeps the
  // products out of a common schedule).
  const bool busy = D == 128 || W == 8 || c0 < cols;
  // A step: the weights of tile t, with which tile t + 1 (fetched a step earlier) is
  // unpacked, the tables of t + 2 are written, and tile t + 2 and the scale words of t + 3
  // are fetched; then the matrix products of the scores of t + 1 and of the values of t.
  // (Tiles from t1 on too, pages past the last as the last: nothing uses them, and the
  // loop has no conditions.)
  auto step = [&](uint32_t t, auto masked) __attribute__((always_inline)) {
    const Pages p2 = page_ids(t + 2), p3 = page_ids(t + 3);
    stage_in(t + 1, raw);
    fetch(p2, raw);
    if (busy) {
      if constexpr (kTight) products(t);
      weights(t, masked);
    } else if (__builtin_amdgcn_readfirstlane(*(const uint32_t*)(table(t) + L::kMisc + 4)) & kHasWide) {
      near = false;
    }
    write_table(t + 2, words);
    fetch_words(p3, words);
    if (((t - t0) & 31) == 16 && wave == W - 1) load_ids(t + 16);  // (in use from 13 steps on)
    if (busy && kTight) add_values(t);
    lds_barrier();
    if (busy && !kTight) {
      products(t + 1);
      add_values(t);
    }
  };
  if (busy && !kTight) products(t0);
  // Tiles below full_end are visible to every column of the wave.
  const uint32_t first_row = min(c0, cols - 1) / gh;
  const uint32_t full_end = min(max(min(args.start + first_row + 1, sq.len) / 32, t0), t1);
  uint32_t t = t0;
  for (; t < full_end && __builtin_expect_with_probability(near, true, 1.0); ++t) step(t, BoolTag<false>{});
  for (; t < t1 && __builtin_expect_with_probability(near, true, 1.0); ++t) step(t, BoolTag<true>{});
  if (__builtin_expect_with_probability(!near, false, 1.0)) return false;

  const float l_tot = l_lane + __shfl_xor(l_lane, 32);
  const float unit = t0 < t1 ? *(const float*)(table(t1 - 1) + L::kMisc) : 1.0f;
  if (!place.col_ok) return true;
  if (leaves_partials(args, place)) {
    // Partials as in decode, row by row: O [row][split][H][D], then (m, l): here O over
    // its own sum, whose logarithm goes into m, so that it stays finite.
    const size_t pr = ((size_t)row * args.splits + place.split) * H + head;
    float* po = args.partials + pr * D;
    const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
#pragma unroll
    for (int db = 0; db < kDB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(floatx4*)(po + 32 * db + 8 * g + 4 * hf) =
            floatx4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]} * inv * unit;
    if (hf == 0)
      *(float2*)(args.partials + (size_t)args.part_rows * H * D + pr * 2) =
          l_tot == 0.0f ? float2{-FLT_MAX, 0.0f} : float2{m_run + log2f(l_tot), 1.0f};
    return true;
  }
  const float inv = 1.0f / l_tot;
  const size_t obase = ((size_t)row * H + head) * dr;
  if (args.out8) {  // 8-byte accesses: dr % 8 == 0, o and gate aligned
    u32x2 gt[kDB][4];
    if (args.gate) {
#pragma unroll
      for (int i = 0; i < kDB * 4; ++i) {
        const uint32_t d0 = 8 * i + 4 * hf;
        if (d0 < dr) gt[i >> 2][i & 3] = *(const u32x2*)(args.gate + obase + d0);
      }
    }
#pragma unroll
    for (int i = 0; i < kDB * 4; ++i) {
      const uint32_t d0 = 8 * i + 4 * hf;
      if (d0 >= dr) continue;
      const int db = i >> 2, g = i & 3;
      const floatx4 v = floatx4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]} * inv * unit;
      *(u32x2*)(args.o + obase + d0) = args.gate ? gated_bf16x4(v, gt[db][g]) : bf16x4_of(v);
    }
  } else {
#pragma unroll 1
    for (int e = 0; e < 16; ++e)
#pragma unroll
      for (int db = 0; db < kDB; ++db) {
        const uint32_t d = 32 * db + 8 * (e >> 2) + 4 * hf + (e & 3);
        if (d >= dr) continue;
        float v = o[db][e] * inv * unit;
        if (args.gate) v *= gate_sigmoid(bf16_to_f32(args.gate[obase + d]));
        args.o[obase + d] = f32_to_bf16(v);
      }
  }
  return true;
}

template <int D, int W>
__global__ __launch_bounds__(64 * W, attn_prefill_waves(D, W)) void q4kv_prefill_kernel(Q4KvPrefillArgs args) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[PrefillLds<D, W>::kBytes];
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (__builtin_expect_with_probability(prefill_block<D, W>(args, lds, wave), true, 1.0)) return;
  prefill_far<D, W>(args, wave);
}

template <int D, int W>
hipError_t launch_prefill(const AttnArgs& a, hipStream_t st) {
  const uint32_t cols = a.rows * (a.heads / a.kv_heads);
  const uint32_t blocks = (cols + 32 * W - 1) / (32 * W);
  uint32_t units = blocks * a.splits;
  Q4KvPrefillArgs args{};
  (AttnArgs&)args = a;
  if (a.split_tiles) {
    // (A workgroup that only ends would not do: they are dealt to the shader engines in
    // turn, and some of those would get few others.)
    units = 0;
    for (uint32_t s = 0, first = 0; s < (uint32_t)kMaxBlockSplits; ++s) {
      while (first < blocks && s > 0 &&
             prefill_block_splits(prefill_tiles(first, 32 * W, cols, a.heads / a.kv_heads, a.start, a.seqs[0].len),
                                  a.split_tiles, a.splits) <= s)
        ++first;
      args.split_begin[s] = s < a.splits ? units : ~0u;
      units += blocks - first;
    }
  }
  hipLaunchKernelGGL((q4kv_prefill_kernel<D, W>), dim3(units * a.kv_heads), dim3(64 * W), 0, st, args);
  if (a.splits > 1) launch_attn_combine(combine_args(a), st);
  return hipGetLastError();
}

template <int D>
hipError_t launch_prefill_d(const AttnArgs& a, hipStream_t st) {
  return a.wg_waves == 8 ? launch_prefill<D, 8>(a, st) : launch_prefill<D, 4>(a, st);
}

template <int D>
hipError_t launch_decode_d(const Q4KvArgs& a, uint32_t units, bool need_combine, hipStream_t st) {
  if (a.wg_waves == 8)
    hipLaunchKernelGGL((q4kv_decode_kernel<D, 8>), dim3(units), dim3(512), 0, st, a);
  else
    hipLaunchKernelGGL((q4kv_decode_kernel<D, 4>), dim3(units), dim3(256), 0, st, a);
  if (need_combine) launch_attn_combine(combine_args(a), st);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_q4kv_prefill(const AttnArgs& a, hipStream_t st) {
  // (Blocks of one split leave partials too where there is a gate.)
  if (a.splits == 0 || ((a.splits > 1 || a.split_tiles) && !a.partials)) return hipErrorInvalidValue;
  switch (a.head_dim_pad) {
    case 64: return launch_prefill_d<64>(a, st);
    case 128: return launch_prefill_d<128>(a, st);
    case 256: return launch_prefill_d<256>(a, st);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_q4kv_decode(const Q4KvArgs& a, uint32_t units, bool need_combine, hipStream_t st) {
  if (need_combine && !a.partials) return hipErrorInvalidValue;
  switch (a.head_dim_pad) {
    case 64: return launch_decode_d<64>(a, units, need_combine, st);
    case 128: return launch_decode_d<128>(a, units, need_combine, st);
    case 256: return launch_decode_d<256>(a, units, need_combine, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace qm
