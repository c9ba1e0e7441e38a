// Latent attention, absorbed form: the queries go into the latent space
// (q_nope W_uk), attend over the 8-bit cache as over one shared key and value
// per token, and the sums of latents come out through W_uv.  For decode and
// for few rows: a token costs 584 bytes (rank 512) whatever the heads.
//
// Four launches: latent_query_kernel (which also appends the new rows),
// latent_attn_kernel (split over the cache's length), latent_join_kernel,
// latent_up_kernel.
#include <float.h>

#include <type_traits>

#include "latent.h"
#include "latent_append.h"
#include "latent_device.h"

namespace qm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoMax = -1e30f;  // running maximum before the first visible token

// ---------------------------------------------------------------------------
// New rows into the cache, queries into the latent space
// ---------------------------------------------------------------------------
// The first workgroups append the call's rows (four a workgroup); the others
// form qa[h][r] = sum_d q_nope[h][d] W_uk[h][d][r] and write it, and apart from
// it the rotated part, as 16-bit integers in two 8-bit digits: q = qs * (256 hi +
// lo), hi in -127..127, lo in -128..127.  The scores are then whole-number
// products with the cache's codes on the i8 matrix cores, exact but for this
// rounding, and the codes need no conversion.  qs = bound / 32512: for qa the
// bound is |q_nope| times the head's largest column norm of W_uk (usually 2 or 3
// times the row's largest element, so qa is rounded to about 2^-15 of that,
// where bf16 would round each element to 2^-8), which lets the row be cut over
// workgroups; for the rotated part it is its largest element.  A row with a NaN
// or an infinity gets a NaN scale, which its scores keep.
//
// Workgroup = (16 rows, head, 128 latent elements), a wave 32 of them: D = W
// (rows) x queries (columns), so a lane holds four consecutive elements of a
// row.  One token of 32 heads (4 MB of weights) is bound by latency: 128
// workgroups of one round trip each.
__device__ __forceinline__ void two_digits(float v, float s, bool skip, int at, uint32_t* hi, uint32_t* lo) {
  const int q = skip ? 0 : (int)rintf(fminf(fmaxf(v / s, -32512.0f), 32512.0f));
  const int h8 = (q + 128) >> 8;
  *hi |= ((uint32_t)h8 & 255u) << (8 * at);
  *lo |= ((uint32_t)(q - 256 * h8) & 255u) << (8 * at);
}

template <int RP>
__global__ __launch_bounds__(256) void latent_query_kernel(LatentAttnArgs a, uint32_t append_blocks) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (blockIdx.x < append_blocks) {
    const uint32_t item = blockIdx.x * 4 + wave;
    if (item >= a.rows) return;
    const LatentSeq& sq = a.seqs[a.decode ? item : 0];
    latent_append_row(a.new_rows, sq.rows, sq.start + (a.decode ? 0 : item), item, lane);
    return;
  }
  const uint32_t H = a.d.heads, nope = a.d.nope, qw = nope + a.d.rope, np = a.d.nope_pad;
  uint32_t unit = blockIdx.x - append_blocks;
  const uint32_t chunk = unit % (RP / 128);
  unit /= RP / 128;
  const uint32_t h = unit % H, m0 = unit / H * 16;
  const uint32_t n = lane & 15, kq = lane >> 4, m = m0 + n;
  const bool live = m < a.rows;
  const uint16_t* down = a.down + ((size_t)h * RP + chunk * 128 + wave * 32) * np;
  const uint16_t* qrow = a.q + ((size_t)min(m, a.rows - 1) * H + h) * qw;
  u32x4 x[4], w[2][4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const uint32_t k = 32 * s + 8 * kq;
    x[s] = k < nope && live ? *(const u32x4*)(qrow + k) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < 2; ++t)
      w[t][s] = 32u * s < np ? *(const u32x4*)(down + (size_t)(16 * t + n) * np + k) : u32x4{0, 0, 0, 0};
  }
  // |q|, scaled by a power of two against overflow; the largest absolute value
  // as bits, where NaN and infinity come out on top.
  uint32_t top = 0;
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int k = 0; k < 4; ++k) top = max(top, max(x[s][k] & 0x7FFF0000u, (x[s][k] << 16) & 0x7FFF0000u));
  top = max(top, (uint32_t)__shfl_xor((int)top, 16));
  top = max(top, (uint32_t)__shfl_xor((int)top, 32));
  const bool bad = top >= 0x7F800000u;
  const uint32_t e = min(max(top & 0x7F800000u, 0x01000000u), 0x7E000000u);
  const float down_scale = __uint_as_float(0x7F000000u - e);
  float ss = 0.0f;
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float lo = __uint_as_float(x[s][k] << 16) * down_scale;
      const float hi = __uint_as_float(x[s][k] & 0xFFFF0000u) * down_scale;
      ss = fmaf(lo, lo, fmaf(hi, hi, ss));
    }
  ss += __shfl_xor(ss, 16);
  ss += __shfl_xor(ss, 32);
  const float qs = fmaxf(sqrtf(ss) * a.wnorm[h] / 32512.0f * __uint_as_float(e), FLT_MIN);

  floatx4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int t = 0; t < 2; ++t) acc[t] = mfma16x16x32(w[t][s], x[s], acc[t]);
  const float nan = __uint_as_float(0x7FC00000u);
  if (live) {
    const uint32_t c = a.decode ? h : m * H + h, col = c % kLatentCols;
    const size_t block = a.seqs[a.decode ? m : 0].block_begin + c / kLatentCols;
    uint8_t* to = a.digits + block * latent_digit_bytes(RP) + col * 32;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t hi = 0, lo = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) two_digits(acc[t][i], qs, bad, i, &hi, &lo);
      // Piece of 16 elements 16 t of the wave's 32: steps are 32 elements, halves 16.
      uint8_t* at = to + ((chunk * 4 + wave) * 64 + t * 32) * 32 + 4 * kq;
      *(uint32_t*)at = hi;
      *(uint32_t*)(at + 16) = lo;
    }
    if (chunk == 0 && wave == 0 && kq == 0) a.qscale[(block * kLatentCols + col) * 2] = bad ? nan : qs;
  }
  if (chunk != 0) return;
  // The rotated part: 16 threads a row, 4 elements each.
  const uint32_t t = threadIdx.x & 15, mk = m0 + (threadIdx.x >> 4);
  const uint16_t* key = a.q + ((size_t)min(mk, a.rows - 1) * H + h) * qw + nope;
  float k[4];
  uint32_t top_key = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    k[i] = 4 * t + i < a.d.rope ? bf16_to_f32(key[4 * t + i]) : 0.0f;
    top_key = max(top_key, __float_as_uint(k[i]) & 0x7FFFFFFFu);
  }
#pragma unroll
  for (int s = 1; s < 16; s *= 2) top_key = max(top_key, (uint32_t)__shfl_xor((int)top_key, s));
  if (mk >= a.rows) return;
  const float ks = fmaxf(__uint_as_float(top_key) / 32512.0f, FLT_MIN);
  const bool bad_key = top_key >= 0x7F800000u;
  const uint32_t c = a.decode ? h : mk * H + h, col = c % kLatentCols;
  const size_t block = a.seqs[a.decode ? mk : 0].block_begin + c / kLatentCols;
  uint32_t hi = 0, lo = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) two_digits(k[i], ks, bad_key, i, &hi, &lo);
  uint8_t* at = a.digits + block * latent_digit_bytes(RP) +
                ((RP / 32 + t / 8) * 64 + (t / 4 % 2) * 32 + col) * 32 + 4 * (t % 4);
  *(uint32_t*)at = hi;
  *(uint32_t*)(at + 16) = lo;
  if (t == 0) a.qscale[(block * kLatentCols + col) * 2 + 1] = bad_key ? nan : ks;
}

// ---------------------------------------------------------------------------
// Attention over the cache
// ---------------------------------------------------------------------------
// Workgroup = (32 NC columns, a share of the cache's 64-token tiles), eight waves,
// one workgroup a CU.  A column is a head of a row.  The tiles' bytes stream into
// an LDS ring by buffer->LDS DMA and are read from there as they lie:
//   scores   S^T[token][column] = codes . (hi, lo) on v_mfma_i32_32x32x32_i8.  A
//            wave has a column block, 32 of the tokens and a part of the latent
//            (a half, or a quarter with one column block); the parts exchange
//            their whole numbers through LDS and each finishes a share of the
//            tokens, where the token's and the column's scales come in in fp32.
//            Cutting the latent keeps the queries in registers once.
//   softmax  online, in fp32: p = 2^(s - ref), ref a column's maximum less 6,
//            moved (and the sums rescaled) only when a maximum passes ref + 14, so
//            p stays below 2^14 and what is 2^-20 of the largest is still a normal
//            fp16.  The waves compute p with the ref they have and publish it with
//            their maxima; where one passes, all see it behind the same barrier
//            and do it again.
//   sums     O^T[latent element][column] += codes^T P'^T on
//            v_mfma_f32_32x32x16_f16, a wave an eighth of the latent: P' = token
//            scale * p / 2^w, w moved like ref with the largest p * token scale;
//            rounded to fp16 (2^-11 of each term, where bf16 would be 2^-8), the
//            codes exact.  The codes' operand comes by transposing
//            reads; its conversion is shared by the wave's columns.
// Two barriers a tile: the scores' exchange, and P'.
template <int RP, int NC>
struct AbsorbedLds {
  static constexpr int kChunks = RP / 16;  // 16-byte pieces of a latent
  static constexpr int kLat = kLatentTile * RP, kKey = kLatentTile * (int)kLatentRope, kScale = kLatentTile * 8;
  static constexpr int kTileBytes = kLat + kKey + kScale;
  static constexpr int kRing = 3;
  static constexpr int kParts = 4 / NC;       // of the contraction
  static constexpr int kShare = 16 / kParts;  // scores of a lane that a wave finishes
  static constexpr int kExchange = NC == 1 ? 32768 : 16384;
  static constexpr int kP = NC * 4096, kMax = 2 * kParts * NC * 32 * 8;
  static constexpr int kBytes = kRing * kTileBytes + kExchange + kP + kMax;
  static constexpr int kDma = RP / 128 + 2;  // DMA instructions of a wave and tile
};

// Order of a token's 16-byte pieces in LDS: piece j at j ^ swizzle(token).  Both
// the reads of one piece of 8 consecutive tokens and those of the 8 tokens of a
// transposing read (0..3, 8..11 or 4..7, 12..15) fall on different banks.
__device__ __forceinline__ constexpr uint32_t lat_swizzle(uint32_t tok) {
  return (tok & 3) | ((((tok >> 2) ^ (tok >> 3)) & 1) << 2);
}

template <int RP, int NC>
__global__ __launch_bounds__(512, 2) void latent_attn_kernel(LatentAttnArgs a) {
  using L = AbsorbedLds<RP, NC>;
  constexpr int CH = L::kChunks, kParts = L::kParts, kShare = L::kShare;
  constexpr int kLatSteps = RP / 32 / kParts;       // a wave's
  constexpr int kAll = RP / 32, kBlocks = (kAll + 7) / 8;  // blocks of 32 latent elements: all, a wave's
  constexpr uint32_t kStride = RP + kLatentRope, kCols = 32 * NC;
  __shared__ __attribute__((aligned(16))) uint8_t lds[L::kBytes];
  uint8_t* const exchange = lds + L::kRing * L::kTileBytes;
  uint8_t* const pbuf = exchange + L::kExchange;
  float2* const maxima = (float2*)(pbuf + L::kP);  // [token block][part][column]: of s, of p * token scale
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t col = lane & 31, half = lane >> 5;
  const uint32_t unit = blockIdx.x, H = a.d.heads;
  uint32_t b = 0;
  while (b + 1 < a.n_seqs && unit >= a.seqs[b + 1].unit_begin) ++b;
  const LatentSeq& sq = a.seqs[b];
  const uint32_t cols = a.decode ? H : a.rows * H;
  const uint32_t groups = (cols + kCols - 1) / kCols;
  const uint32_t local = unit - sq.unit_begin, cg = local % groups, split = local / groups;
  // The wave's scores: a block of tokens, a column block, a part of the contraction.
  const uint32_t tb = wave & 1, my_block = NC == 1 ? 0 : (wave >> 1) & 1, part = wave / (2 * NC);
  // Tokens that a column sees: up to its own row.
  const uint32_t c_first = cg * kCols, c_last = min(c_first + kCols, cols) - 1, c = c_first + 32 * my_block + col;
  const uint32_t lim_min = sq.start + c_first / H + 1, lim_max = sq.start + c_last / H + 1;
  const uint32_t limit = c <= c_last ? sq.start + c / H + 1 : 0;
  const uint32_t tiles = (lim_max + kLatentTile - 1) / kLatentTile;
  const uint32_t t_begin = split * a.tiles_per_split, t_end = min(tiles, t_begin + a.tiles_per_split);

  // A tile's bytes, an eighth a wave: pieces of 1 KB of the latents, 512 bytes of
  // the shared keys, 64 of the scales.
  auto issue = [&](uint32_t tile, uint32_t slot) __attribute__((always_inline)) {
    uint8_t* to = lds + slot * L::kTileBytes;
    const auto rows = latent_rsrc(sq.rows.codes + (size_t)tile * kLatentTile * kStride, kLatentTile * kStride);
#pragma unroll
    for (int i = 0; i < RP / 128; ++i) {
      const uint32_t p0 = (wave * (RP / 128) + i) * 64;
      if constexpr (64 % CH == 0) {  // whole tokens: piece j of token p0 / CH + lane / CH
        const uint32_t t0 = lane / CH, j = (lane % CH) ^ lat_swizzle(t0) ^ lat_swizzle(p0 / CH);
        latent_dma16(rows, to + p0 * 16, t0 * kStride + j * 16, p0 / CH * kStride);
      } else {
        const uint32_t tok = (p0 + lane) / CH, j = ((p0 + lane) % CH) ^ lat_swizzle(tok);
        latent_dma16(rows, to + p0 * 16, tok * kStride + j * 16, 0);
      }
    }
    if (lane < 32) {  // token 8 wave + lane / 4, piece (lane % 4) ^ (token / 2 % 4)
      const uint32_t tok = lane / 4;
      latent_dma16(rows, to + L::kLat + wave * 512, tok * kStride + RP + (((lane & 3) ^ ((tok >> 1) & 3)) * 16),
                   8 * wave * kStride);
    }
    const auto scales = latent_rsrc(sq.rows.scales + (size_t)tile * kLatentTile * 2, kLatentTile * 8);
    if (lane < 16) latent_dma4(scales, to + L::kLat + L::kKey + wave * 64, wave * 64 + lane * 4);
  };
#pragma unroll
  for (int i = 0; i < L::kRing - 1; ++i)
    if (t_begin + i < t_end) issue(t_begin + i, i);

  // (A group's last block may be one that does not exist; its columns have no tokens.)
  const size_t block = sq.block_begin + min(cg * NC + my_block, (cols - 1) / 32);
  u32x4 qhi[kLatSteps + 2], qlo[kLatSteps + 2];  // the shared key's last
  {
    const uint8_t* dg = a.digits + block * latent_digit_bytes(RP) + lane * 32;
#pragma unroll
    for (int s = 0; s < kLatSteps + 2; ++s) {
      const uint32_t step = s < kLatSteps ? part * kLatSteps + s : kAll + s - kLatSteps;
      qhi[s] = *(const u32x4*)(dg + step * 2048);
      qlo[s] = *(const u32x4*)(dg + step * 2048 + 16);
    }
  }
  const float2 qs = limit ? *(const float2*)(a.qscale + (block * kLatentCols + col) * 2) : float2{0.0f, 0.0f};
  const float lat_scale = qs.x * a.scale * kLog2e, key_scale = qs.y * a.scale * kLog2e;

  // LDS offsets of this lane: codes of its token (score operands) and of the 8
  // tokens of a transposing read.
  const uint32_t tok0 = 32 * tb + col;
  const uint32_t trow = (lane & 15) >> 1, vtok = 4 * half + (trow < 4 ? trow : trow + 4);
  const uint32_t ka = tok0 * RP + ((half ^ lat_swizzle(tok0)) * 16);
  const uint32_t kk = tok0 * kLatentRope + ((half ^ ((tok0 >> 1) & 3)) * 16);
  const uint32_t va = vtok * RP + ((((lane >> 4) & 1) ^ lat_swizzle(vtok)) * 16) + 8 * (lane & 1);

  floatx16 O[kBlocks][NC];
#pragma unroll
  for (int i = 0; i < kBlocks; ++i)
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int j = 0; j < 16; ++j) O[i][n][j] = 0.0f;
  float mref[NC], w2[NC], l = 0.0f;  // ref, w
#pragma unroll
  for (int n = 0; n < NC; ++n) mref[n] = kNoMax, w2[n] = 0.0f;

  latent_wait_vmcnt<0>();
  lds_barrier();
  uint32_t slot = 0;
  for (uint32_t tile = t_begin; tile < t_end; ++tile) {
    const uint8_t* lat = lds + slot * L::kTileBytes;
    const uint8_t* key = lat + L::kLat;
    const float* scales = (const float*)(key + L::kKey);

    // The wave's part of the latent's products, then all of the shared key's: 256
    // hi + lo in whole numbers (at most 512 * 127 * 127 * 256 + 512 * 128 * 127 <
    // 2^31).
    int kdot[kShare], ldot[kShare];
    {
      intx16 hi = {}, lo = {};
#pragma unroll
      for (int s = 0; s < kLatSteps; ++s) {
        const uint32_t step = part * kLatSteps + s;
        const u32x4 kf = *(const u32x4*)(lat + (ka ^ ((step & 3) * 32)) + (step >> 2) * 128);
        hi = mfma32x32x32_i8(kf, qhi[s], hi);
        lo = mfma32x32x32_i8(kf, qlo[s], lo);
      }
      // Shares of the other parts' waves: [column block][token block][to][from], 64
      // lanes x 4 scores a KB.
      const uint32_t tile_at = (my_block * 2 + tb) * kParts;
#pragma unroll
      for (int q = 0; q < kParts; ++q) {
        int d[kShare];
#pragma unroll
        for (int i = 0; i < kShare; ++i) d[i] = (hi[q * kShare + i] << 8) + lo[q * kShare + i];
        if (part == (uint32_t)q) {
#pragma unroll
          for (int i = 0; i < kShare; ++i) ldot[i] = d[i];
        } else {
#pragma unroll
          for (int i = 0; i < kShare / 4; ++i) {
            const uint32_t at = NC == 1 ? (tile_at + q) * 4 + part : (tile_at + q) * 2 + i;
            *(intx4*)(exchange + at * 1024 + lane * 16) = intx4{d[4 * i], d[4 * i + 1], d[4 * i + 2], d[4 * i + 3]};
          }
        }
      }
      __asm__ volatile("" ::: "memory");  // not both products' sums at once: registers
      intx16 khi = {}, klo = {};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const u32x4 kf = *(const u32x4*)(key + (kk ^ (s * 32)));
        khi = mfma32x32x32_i8(kf, qhi[kLatSteps + s], khi);
        klo = mfma32x32x32_i8(kf, qlo[kLatSteps + s], klo);
      }
#pragma unroll
      for (int q = 0; q < kParts; ++q)
        if (part == (uint32_t)q)
#pragma unroll
          for (int i = 0; i < kShare; ++i) kdot[i] = (khi[q * kShare + i] << 8) + klo[q * kShare + i];
      lds_barrier();  // scores exchanged; every wave is done with the tile before
      if (tile + L::kRing - 1 < t_end) issue(tile + L::kRing - 1, slot == 0 ? L::kRing - 1 : slot - 1);
#pragma unroll
      for (int f = 0; f < (NC == 1 ? 4 : 2); ++f) {
        if (NC == 1 && part == (uint32_t)f) continue;
        const uint32_t at = NC == 1 ? (tile_at + part) * 4 + f : (tile_at + part) * 2 + f;
        const intx4 v = *(const intx4*)(exchange + at * 1024 + lane * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) ldot[(NC == 1 ? 0 : 4 * f) + j] += v[j];
      }
    }

    // The wave's share: scores i of a lane are tokens 8 (i / 4) + 4 half + i % 4 of
    // its token block, its own from part * kShare on.
    const uint32_t first = part * kShare;
    float S[kShare], ts[kShare];
#pragma unroll
    for (int g = 0; g < kShare / 4; ++g) {
      const float* at = scales + tb * 64 + (2 * (first / 4 + g) + half) * 8;
      const floatx4 s0 = *(const floatx4*)at, s1 = *(const floatx4*)(at + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = 4 * g + j;
        ts[i] = j < 2 ? s0[2 * j] : s1[2 * j - 4];
        S[i] = fmaf((float)ldot[i], ts[i] * lat_scale, (float)kdot[i] * ((j < 2 ? s0[2 * j + 1] : s1[2 * j - 3]) * key_scale));
      }
    }
    const bool whole = (tile + 1) * kLatentTile <= lim_min && c_last - c_first == kCols - 1;
    if (!whole) {
#pragma unroll
      for (int i = 0; i < kShare; ++i) {
        const uint32_t tok = tile * kLatentTile + 32 * tb + 8 * (first / 4 + i / 4) + 4 * half + i % 4;
        S[i] = tok < limit ? S[i] : -INFINITY;
        ts[i] = tok < limit ? ts[i] : 0.0f;  // nothing of it, not even a scale that is no number
      }
    }
    float top = S[0];
#pragma unroll
    for (int i = 1; i < kShare; ++i) top = fmaxf(top, S[i]);
    top = halves_max(top);
    const uint32_t at_max = (tb * kParts + part) * kCols + 32 * my_block + col;
    float sum, top_pt;
    auto publish = [&]() __attribute__((always_inline)) {
      float p[kShare];
      const bool lower = NC == 1 || my_block == 0;
      const float ref = lower ? mref[0] : mref[NC - 1], unit = __builtin_amdgcn_exp2f(-(lower ? w2[0] : w2[NC - 1]));
      sum = top_pt = 0.0f;
#pragma unroll
      for (int i = 0; i < kShare; ++i) {
        const float e = __builtin_amdgcn_exp2f(S[i] - ref);
        sum += e;
        p[i] = e * ts[i] * unit;
        top_pt = fmaxf(top_pt, p[i]);
      }
      // Pairs in the order of bytes_to_f16; scores 8 u .. 8 u + 7 are contraction block u.
      uint8_t* to = pbuf + (tb * NC + my_block) * 2048 + lane * 16;
      if constexpr (NC == 1)
        *(u32x2*)(to + (part / 2) * 1024 + (part % 2) * 8) = u32x2{to_f16x2(p[0], p[2]), to_f16x2(p[1], p[3])};
      else
        *(u32x4*)(to + part * 1024) =
            u32x4{to_f16x2(p[0], p[2]), to_f16x2(p[1], p[3]), to_f16x2(p[4], p[6]), to_f16x2(p[5], p[7])};
    };
    publish();
    top_pt = halves_max(top_pt);
    if (half == 0) maxima[at_max] = float2{top, top_pt};
    if (tile + 2 < t_end) latent_wait_vmcnt<L::kDma>();  // the next tile's bytes
    else latent_wait_vmcnt<0>();
    lds_barrier();  // P', the maxima and the next tile are in LDS
    bool passed = false;
    float tops[NC];
    auto read_maxima = [&](int n, float* y) __attribute__((always_inline)) {
      float2 m = maxima[32 * n + col];
#pragma unroll
      for (int q = 1; q < 2 * kParts; ++q) {
        const float2 v = maxima[q * kCols + 32 * n + col];
        m.x = fmaxf(m.x, v.x), m.y = fmaxf(m.y, v.y);
      }
      *y = m.y;
      return m.x;
    };
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      float pt;
      tops[n] = read_maxima(n, &pt);
      passed = passed || tops[n] > mref[n] + 14.0f || pt > 16384.0f;
    }
    if (__any(passed)) {  // the same in every wave
      float m[NC];
#pragma unroll
      for (int n = 0; n < NC; ++n) m[n] = fmaxf(mref[n], tops[n] - 6.0f);
      // log2(p * token scale) with the new ref: the waves' maxima again.
      const float own = NC == 1 || my_block == 0 ? m[0] : m[NC - 1];
      float top_w = -INFINITY;
#pragma unroll
      for (int i = 0; i < kShare; ++i) top_w = fmaxf(top_w, S[i] - own + __log2f(ts[i]));
      top_w = halves_max(top_w);
      lds_barrier();
      if (half == 0) maxima[at_max].y = top_w;
      lds_barrier();
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        float w;
        (void)read_maxima(n, &w);
        const float moved = mref[n] - m[n];
        w = fmaxf(fmaxf(w2[n] + moved, w - 6.0f), -100.0f);  // 2^-w stays a number
        const float f = __builtin_amdgcn_exp2f(moved + (w2[n] - w));
        if (NC == 1 || my_block == (uint32_t)n) l *= __builtin_amdgcn_exp2f(moved);
        mref[n] = m[n];
        w2[n] = w;
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) O[i][n][j] *= f;
      }
      publish();
      lds_barrier();
    }
    l += sum;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        u32x4 p[NC];
#pragma unroll
        for (int n = 0; n < NC; ++n) p[n] = *(const u32x4*)(pbuf + ((t * NC + n) * 2 + u) * 1024 + lane * 16);
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) {
          const uint32_t rb = wave + 8 * i;
          if (kAll % 8 != 0 && rb >= kAll) break;
          const u32x4 v = bytes_to_f16(lds_read_tr8(lat + (va ^ ((rb & 3) * 32)) + (rb >> 2) * 128 + (32 * t + 16 * u) * RP));
#pragma unroll
          for (int n = 0; n < NC; ++n) O[i][n] = mfma32x32x16_f16(v, p[n], O[i][n]);
        }
      }
    slot = slot + 1 == L::kRing ? 0 : slot + 1;
  }

  // The columns' softmax sums from the other waves, and the sums of latents as the
  // lanes hold them (1 KB a store; the join reads them likewise).
  l = halves_sum(l);
  lds_barrier();
  if (half == 0) maxima[(tb * kParts + part) * kCols + 32 * my_block + col].x = l;
  lds_barrier();
  float* out = a.partials + (size_t)unit * kCols * RP;
  float* ml = a.partials + (size_t)a.units * kCols * RP + (size_t)unit * kCols * 2;
  if (wave < NC && half == 0) {
    float total = 0.0f;
#pragma unroll
    for (int q = 0; q < 2 * kParts; ++q) total += maxima[q * kCols + 32 * wave + col].x;
    *(float2*)(ml + (32 * wave + col) * 2) = float2{wave == 0 ? mref[0] : mref[NC - 1], total};
  }
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    if (c_first + 32 * n > c_last) break;
    const float f = __builtin_amdgcn_exp2f(w2[n]);
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) {
      const uint32_t rb = wave + 8 * i;
      if (kAll % 8 != 0 && rb >= kAll) break;
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(floatx4*)(out + (((size_t)n * kAll + rb) * 4 + g) * 256 + lane * 4) =
            floatx4{O[i][n][4 * g] * f, O[i][n][4 * g + 1] * f, O[i][n][4 * g + 2] * f, O[i][n][4 * g + 3] * f};
    }
  }
}

// ---------------------------------------------------------------------------
// Joining the splits, and out of the latent space
// ---------------------------------------------------------------------------
// Workgroup = (32 columns, 8 latent elements: one store of the attention's): the
// splits' sums weighted by 2^(m - M), a wave every sixteenth split, added in
// wave order, divided by the joined softmax sum and written as bf16 and the bf16
// of what that leaves (2^-17 in all), the operands of the product with W_uv.
template <int RP, int NC>
__global__ __launch_bounds__(1024) void latent_join_kernel(LatentAttnArgs a) {
  constexpr uint32_t kWaves = 16, kCols = 32 * NC;
  __shared__ floatx4 part[kWaves][64];
  __shared__ float2 red[kWaves][32];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31;
  const uint32_t H = a.d.heads, cols = a.decode ? H : a.rows * H, blocks = (cols + 31) / 32;
  const uint32_t piece = blockIdx.x % (RP / 8), block = blockIdx.x / (RP / 8);
  const uint32_t b = a.decode ? block / blocks : 0, cb = block - b * blocks;
  const LatentSeq& sq = a.seqs[b];
  const uint32_t groups = (cols + kCols - 1) / kCols, n = cb % NC;
  const size_t u0 = sq.unit_begin + cb / NC;
  const float* ml = a.partials + (size_t)a.units * kCols * RP;
  const float* o = a.partials + ((size_t)n * (RP / 8) + piece) * 256 + lane * 4;
  // The wave's splits, relative to their own maximum.
  float top = kNoMax, sum = 0.0f;
  floatx4 acc = {0, 0, 0, 0};
#pragma unroll 4
  for (uint32_t s = wave; s < sq.splits; s += kWaves) {
    const size_t u = u0 + (size_t)s * groups;
    const float2 v = *(const float2*)(ml + (u * kCols + 32 * n + col) * 2);
    const floatx4 x = *(const floatx4*)(o + u * kCols * RP);
    const float m = fmaxf(top, v.x), f = __builtin_amdgcn_exp2f(top - m), g = __builtin_amdgcn_exp2f(v.x - m);
    top = m;
    sum = sum * f + v.y * g;
    acc = acc * f + x * g;
  }
  part[wave][lane] = acc;
  if (lane < 32) red[wave][lane] = float2{top, sum};
  __syncthreads();
  if (wave != 0) return;
  float m = kNoMax;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) m = fmaxf(m, red[w][col].x);
  sum = 0.0f;
  acc = floatx4{0, 0, 0, 0};
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) {
    const float f = __builtin_amdgcn_exp2f(red[w][col].x - m);
    sum += red[w][col].y * f;
    acc += part[w][lane] * f;
  }
  const uint32_t c = cb * 32 + col;
  if (c >= cols) return;
  const float r = 1.0f / sum;
  float x[4], y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = acc[i] * r;
    y[i] = x[i] - (float)(__bf16)x[i];
  }
  uint16_t* to = a.mixed + ((size_t)b * cols + c) * 2 * RP + piece * 8 + 4 * (lane >> 5);
  *(u32x2*)to = u32x2{to_bf16x2(x[0], x[1]), to_bf16x2(x[2], x[3])};
  *(u32x2*)(to + RP) = u32x2{to_bf16x2(y[0], y[1]), to_bf16x2(y[2], y[3])};
}

// o[m][h][n] = sum_r mixed[m][h][r] W_uv[h][n][r]: workgroup = (16 rows, head, 32
// outputs), a wave takes a quarter of the latent; the quarters are added in
// order in LDS.
template <int RP>
__global__ __launch_bounds__(256) void latent_up_kernel(LatentAttnArgs a) {
  __shared__ float part[4][16][33];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, kq = lane >> 4;
  const uint32_t H = a.d.heads, vp = a.d.v_pad;
  const uint32_t n0 = blockIdx.x % (vp / 32) * 32, h = blockIdx.x / (vp / 32) % H, m0 = blockIdx.x / (vp / 32) / H * 16;
  if (n0 >= a.d.v) return;
  const uint16_t* up = a.up + ((size_t)h * (a.d.nope_pad + vp) + a.d.nope_pad + n0) * RP + wave * (RP / 4) + 8 * kq;
  const uint16_t* x = a.mixed + ((size_t)min(m0 + n, a.rows - 1) * H + h) * 2 * RP + wave * (RP / 4) + 8 * kq;
  floatx4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
  for (int s = 0; s < RP / 128; ++s) {
    const u32x4 hi = *(const u32x4*)(x + 32 * s), lo = *(const u32x4*)(x + RP + 32 * s);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const u32x4 w = *(const u32x4*)(up + (size_t)(16 * t + n) * RP + 32 * s);
      acc[t] = mfma16x16x32(hi, w, acc[t]);
      acc[t] = mfma16x16x32(lo, w, acc[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][4 * kq + i][16 * t + n] = acc[t][i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t at = i * 256 + threadIdx.x, mm = at / 32, nn = at % 32;
    if (m0 + mm >= a.rows || n0 + nn >= a.d.v) continue;
    const float v = part[0][mm][nn] + part[1][mm][nn] + part[2][mm][nn] + part[3][mm][nn];
    a.o[((size_t)(m0 + mm) * H + h) * a.d.v + n0 + nn] = f32_to_bf16(v);
  }
}

template <int RP, int NC>
hipError_t absorbed(const LatentAttnArgs& a, hipStream_t st) {
  const uint32_t tiles = (a.rows + 15) / 16 * a.d.heads, append_blocks = (a.rows + 3) / 4;
  hipLaunchKernelGGL(latent_query_kernel<RP>, dim3(append_blocks + tiles * (RP / 128)), dim3(256), 0, st, a, append_blocks);
  hipLaunchKernelGGL((latent_attn_kernel<RP, NC>), dim3(a.units), dim3(512), 0, st, a);
  hipLaunchKernelGGL((latent_join_kernel<RP, NC>), dim3(a.blocks * (RP / 8)), dim3(1024), 0, st, a);
  hipLaunchKernelGGL(latent_up_kernel<RP>, dim3(tiles * (a.d.v_pad / 32)), dim3(256), 0, st, a);
  return hipGetLastError();
}
template <int RP>
hipError_t absorbed_cols(const LatentAttnArgs& a, hipStream_t st) {
  return a.group_cols == 32 ? absorbed<RP, 1>(a, st) : absorbed<RP, 2>(a, st);
}

}  // namespace

hipError_t launch_latent_absorbed(const LatentAttnArgs& a, hipStream_t st) {
  switch (a.d.rank_pad) {
    case 128: return absorbed_cols<128>(a, st);
    case 256: return absorbed_cols<256>(a, st);
    case 384: return absorbed_cols<384>(a, st);
    default: return absorbed_cols<512>(a, st);
  }
}

}  // namespace qm
