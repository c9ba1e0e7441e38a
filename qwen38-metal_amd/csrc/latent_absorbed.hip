// Latent attention, absorbed form: the queries go into the latent space
// (q_nope W_uk), attend over the 8-bit cache as over one shared key and value
// per token, and the sums of latents come out through W_uv.  For decode and
// for few rows: a token costs 584 bytes (rank 512) whatever the heads.
//
// Four launches: latent_query_kernel (which also appends the new rows),
// latent_attn_kernel (split over the cache's length), latent_join_kernel,
// latent_up_kernel.
#include <float.h>

#include <algorithm>
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
// or an infinity gets a NaN scale, which its scores keep; so does every row of a
// head whose W_uk holds one (its norm is no finite number).
//
// Workgroup = (16 rows, head, 128 latent elements), a wave 32 of them: D = W
// (rows) x queries (columns), so a lane holds four consecutive elements of a
// row.  One token of 32 heads (4 MB of weights) is bound by latency: 128
// workgroups of one round trip each, 6.8 us with the launch; of 128 heads (17 MB)
// 7.2.
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
    latent_append_rows<1>(a.new_rows, sq.rows, sq.start + (a.decode ? 0 : item), item, item + 1, lane);
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
  const float wnorm = a.wnorm[h];
  const bool bad = top >= 0x7F800000u || !(wnorm <= FLT_MAX);  // (fmaxf below would drop a NaN)
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
  const float qs = fmaxf(sqrtf(ss) * wnorm / 32512.0f * __uint_as_float(e), FLT_MIN);

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
// Workgroup = (32 NC columns, a share of the cache's 32-token blocks), eight waves,
// one workgroup a CU.  A column is a head of a row.  The blocks' bytes stream into
// an LDS ring by buffer->LDS DMA and are read from there as they lie, two blocks
// (64 tokens) at a time:
//   scores   S^T[token][column] = codes . (hi, lo) on v_mfma_i32_32x32x32_i8.  A
//            wave has a block, a column block and a part of the latent (a half, or
//            a quarter with one column block), which keeps the queries in registers
//            once; the parts exchange their whole numbers through LDS and each
//            finishes a share of the tokens,
//   softmax  where the token's and the column's scales come in in fp32; online: p =
//            2^(s - ref), ref a column's maximum less 6, moved (and the sums
//            rescaled) only when a lane's sum of p passes 2^14, so p stays below
//            that and what is 2^-20 of the largest is still a normal fp16.  The
//            waves compute p with the ref they have and publish it; where a sum (or
//            a P', below) passes 2^14, a flag says so behind the same barrier and it
//            is done again; so is, at once, a block that some column does not see
//            whole.
//   sums     O^T[latent element][column] += codes^T P'^T on
//            v_mfma_f32_32x32x16_f16, a wave an eighth of the latent: P' = token
//            scale * p / 2^w, w moved like ref with the largest p * token scale;
//            rounded to fp16 (2^-11 of each term, where bf16 would be 2^-8), the
//            codes exact.  The codes' operand comes by transposing reads; its
//            conversion is shared by the wave's columns.
// Two barriers for 64 tokens.  Between the first (scores exchanged) and the second
// (P' written) the softmax's vector work runs mixed with the latent's part of the
// next scores, behind the second the sums' products and the shared key's part.
//
// With 128 heads and 131072 tokens the loop takes about 4800 cycles for 64 tokens of
// 64 columns, 2304 of them the matrix cores' and as many the vector unit's, which two
// waves a SIMD overlap in part; before it 4 us until queries and first blocks are
// there, behind it 33 MB of partial sums.  54 us in all, 75 MB read (1.4 TB/s).  With
// masks and maxima for every block: 55; with softmax and all products in phases of
// their own: 59; waits of LDS reads for the copies in flight (what the compiler makes
// of its own copy builtin): 71.
template <int RP, int NC>
struct AbsorbedLds {
  static constexpr int kChunks = RP / 16;  // 16-byte pieces of a latent
  static constexpr int kLat = kLatentTile * RP, kKey = kLatentTile * (int)kLatentRope, kScale = kLatentTile * 8;
  static constexpr int kTileBytes = kLat + kKey + kScale;
  static constexpr int kRing = 6;
  static constexpr int kParts = 4 / NC;       // of the contraction
  static constexpr int kShare = 16 / kParts;  // scores of a lane that a wave finishes
  static constexpr int kExchange = NC == 1 ? 32768 : 16384;
  static constexpr int kP = NC * 4096, kMax = 2 * kParts * NC * 32 * 8;
  static constexpr int kKeyDigits = NC * 4096;  // of the queries' rotated part [block][step][hi, lo][lane]
  // The ring last: the others are then in reach of an instruction's offset.
  static constexpr int kAtP = kExchange, kAtMax = kAtP + kP, kAtKeys = kAtMax + kMax, kAtFlag = kAtKeys + kKeyDigits;
  // Registers: with two column blocks and many steps the lower digits of a wave's
  // first steps live here.
  static constexpr int kLowSteps = NC == 2 && RP / 32 / kParts >= 6 ? RP / 32 / kParts / 2 : 0;
  static constexpr int kAtLow = kAtFlag + 16, kLow = kLowSteps * 4096;
  static constexpr int kAtRing = kAtLow + kLow, kBytes = kAtRing + kRing * kTileBytes;
  static_assert(kAtRing < 65536, "the offsets' range");
  static constexpr int kPieces = (RP / 32 + 7) / 8;  // KB of the latents that a wave brings
  static constexpr int kDma = kPieces + 1;           // DMA instructions of a wave and block, at most
};

// Order of a token's 16-byte pieces in LDS: piece j at j ^ swizzle(token).  The
// banks repeat after 16 pieces.  Reads of one piece of 16 consecutive tokens, and
// transposing reads of two adjacent pieces of 8 tokens (0..3, 8..11 or 4..7, 12..15),
// fall on different ones.  Rows of an odd number of 8 pieces (rank_pad 128, 384)
// alternate between the halves by themselves.
template <int CH>
__device__ __forceinline__ constexpr uint32_t lat_swizzle(uint32_t t) {
  const uint32_t b0 = t & 1, b1 = (t >> 1) & 1, b2 = (t >> 2) & 1, b3 = (t >> 3) & 1;
  return CH % 16 == 0 ? b3 | (b0 << 1) | (b1 << 2) | ((b2 ^ b3) << 3) : b2 | (b1 << 1) | ((b2 ^ b3) << 2);
}
// The shared key's four pieces: four tokens to a round of banks.
__device__ __forceinline__ constexpr uint32_t key_swizzle(uint32_t t) { return (t >> 2) & 3; }

template <int RP, int NC>
__global__ __launch_bounds__(512, 2) void latent_attn_kernel(LatentAttnArgs a) {
  using L = AbsorbedLds<RP, NC>;
  constexpr int CH = L::kChunks, kParts = L::kParts, kShare = L::kShare;
  constexpr int kLatSteps = RP / 32 / kParts;       // a wave's
  constexpr int kAll = RP / 32, kBlocks = (kAll + 7) / 8;  // blocks of 32 latent elements: all, a wave's
  constexpr uint32_t kStride = RP + kLatentRope, kCols = 32 * NC;
  __shared__ __attribute__((aligned(16))) uint8_t lds[L::kBytes];
  uint8_t* const exchange = lds;
  uint8_t* const pbuf = lds + L::kAtP;
  float2* const maxima = (float2*)(lds + L::kAtMax);  // [token block][part][column]: of s, of p * token scale
  uint8_t* const key_digits = lds + L::kAtKeys;
  uint32_t* const flag = (uint32_t*)(lds + L::kAtFlag);  // a maximum has passed
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
  // The wave's scores: one of the two blocks, a column block, a part of the contraction.
  const uint32_t tb = wave >> 2, my_block = NC == 1 ? 0 : wave & 1, part = NC == 1 ? wave & 3 : (wave >> 1) & 1;
  // Tokens that a column sees: up to its own row.
  const uint32_t c_first = cg * kCols, c_last = min(c_first + kCols, cols) - 1, c = c_first + 32 * my_block + col;
  const uint32_t lim_max = sq.start + c_last / H + 1;
  const uint32_t tiles = (lim_max + kLatentTile - 1) / kLatentTile;
  const uint32_t t_begin = split * a.tiles_per_split, t_end = min(tiles, t_begin + a.tiles_per_split);
  const uint32_t n = t_begin < t_end ? t_end - t_begin : 0;
  const uint32_t lim_min = min(sq.start + c_first / H + 1, t_end * kLatentTile);
  const uint32_t limit = c <= c_last ? min(sq.start + c / H + 1, t_end * kLatentTile) : 0;

  const int8_t* const codes = sq.rows.codes;
  const float* const row_scales = sq.rows.scales;
  // A block's bytes, in pieces of 1 KB: the latents' over all waves (some twice
  // where eight do not divide them), two of the shared keys, and the scales.
  constexpr bool kAlike = 512 % CH == 0 && 512 / CH % 16 == 0;  // a wave's pieces differ by whole periods of the swizzle
  constexpr int kFrom = kAlike ? 1 : L::kPieces;
  uint32_t from[kFrom];
#pragma unroll
  for (int k = 0; k < kFrom; ++k) {
    const uint32_t at = (wave + 8 * k) % (RP / 32) * 64 + lane, tok = at / CH;
    from[k] = tok * kStride + ((at % CH) ^ lat_swizzle<CH>(tok)) * 16;
  }
  uint32_t from_other = wave == 2 ? lane * 4 : (16 * wave + lane / 4) * kStride + RP + ((lane & 3) ^ key_swizzle(lane / 4)) * 16;
  // Instruction k of kDma; a block that is not `there` reads as zero.
  auto issue = [&](uint32_t tile, uint32_t slot, bool there, int k) __attribute__((always_inline)) {  // slot: its offset
    uint8_t* to = lds + L::kAtRing + slot;
    const auto rows = latent_rsrc(codes + (size_t)tile * kLatentTile * kStride, there ? kLatentTile * kStride : 0);
    if (k < L::kPieces) {
      latent_dma16(rows, to + (wave + 8 * k) % (RP / 32) * 1024, from[kAlike ? 0 : k], kAlike ? k * (512 / CH) * kStride : 0);
    } else if (wave < 2) {
      latent_dma16(rows, to + L::kLat + wave * 1024, from_other, 0);
    } else if (wave == 2) {
      const auto scales = latent_rsrc(row_scales + (size_t)tile * kLatentTile * 2, there ? kLatentTile * 8 : 0);
      latent_dma4(scales, to + L::kLat + L::kKey, from_other);
    }
  };
  // Two blocks before the queries, so that one trip to memory brings both; the next
  // two behind them.
  auto issue_two = [&](uint32_t i) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t j = i; j < i + 2; ++j)
#pragma unroll
      for (int k = 0; k < L::kDma; ++k) issue(t_begin + j, j * L::kTileBytes, t_begin + j < t_end, k);
  };
  issue_two(0);
  // (A group's last block may be one that does not exist; its columns have no tokens.)
  const size_t block = sq.block_begin + min(cg * NC + my_block, (cols - 1) / 32);
  u32x4 qhi[kLatSteps], qlo[kLatSteps];
  {
    const uint8_t* dg = a.digits + block * latent_digit_bytes(RP) + lane * 32;
#pragma unroll
    for (int s = 0; s < kLatSteps; ++s) {
      qhi[s] = *(const u32x4*)(dg + (part * kLatSteps + s) * 2048);
      qlo[s] = *(const u32x4*)(dg + (part * kLatSteps + s) * 2048 + 16);
    }
  }
  const bool brings = tb == 0 && part < 2;  // the rotated part's digits into LDS, once for all waves of a column block
  u32x4 kd[2];
  if (brings) {
    const uint8_t* dg = a.digits + block * latent_digit_bytes(RP) + lane * 32 + (kAll + part) * 2048;
    kd[0] = *(const u32x4*)dg;
    kd[1] = *(const u32x4*)(dg + 16);
  }
  const float2 qs = limit ? *(const float2*)(a.qscale + (block * kLatentCols + col) * 2) : float2{0.0f, 0.0f};
  const float lat_scale = qs.x * a.scale * kLog2e, key_scale = qs.y * a.scale * kLog2e;
  if (brings) {
#pragma unroll
    for (int s = 0; s < L::kLowSteps; ++s) *(u32x4*)(lds + L::kAtLow + s * 4096 + wave * 1024 + lane * 16) = qlo[s];
    uint8_t* to = key_digits + (my_block * 2 + part) * 2048 + lane * 16;
    *(u32x4*)to = kd[0];
    *(u32x4*)(to + 1024) = kd[1];
  }

  // LDS offsets of this lane: codes of its token (score operands) and of the 8
  // tokens of a transposing read.
  const uint32_t trow = (lane & 15) >> 1, vtok = 4 * half + (trow < 4 ? trow : trow + 4);
  const uint32_t ka = col * RP + ((half ^ lat_swizzle<CH>(col)) * 16);
  // Pieces 2 n + .. of a row: the swizzle reaches over 16 (or 8) of them.
  constexpr uint32_t kSpan = CH % 16 == 0 ? 8 : 4;
  auto piece = [](uint32_t at, uint32_t n) __attribute__((always_inline)) {
    return (at ^ ((n % kSpan) * 32)) + n / kSpan * (kSpan * 32);
  };
  const uint32_t va = L::kAtRing + piece(vtok * RP + ((((lane >> 4) & 1) ^ lat_swizzle<CH>(vtok)) * 16) + 8 * (lane & 1), wave);
  static_assert(8 % kSpan == 0, "eight blocks on, the pieces are eight blocks on");

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

  // The wave's part of a block's score products: 256 hi + lo in whole numbers (at
  // most 512 * 127 * 127 * 256 + 512 * 128 * 127 < 2^31) of the latent, and all of
  // the shared key's.
  auto score_step = [](u32x4 kf, u32x4 qh, u32x4 ql, bool start, intx16& hi, intx16& lo) __attribute__((always_inline)) {
    hi = mfma32x32x32_i8(kf, qh, start ? intx16{} : hi);
    lo = mfma32x32x32_i8(kf, ql, start ? intx16{} : lo);
  };
  // The wave's share of its current block, in turn: whole numbers of the
  // latent's and the key's products; then scores (as bits).
  int ldot[kShare] = {}, kdot[kShare] = {};
  auto take_keys = [&](const intx16& hi, const intx16& lo) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < kParts; ++q)
      if (part == (uint32_t)q)
#pragma unroll
        for (int i = 0; i < kShare; ++i) kdot[i] = (hi[q * kShare + i] << 8) + lo[q * kShare + i];
  };
  // Shares of the other parts' waves: [column block][block][to][from], 64 lanes x 4
  // scores a KB.
  const uint32_t tile_at = (my_block * 2 + tb) * kParts * (NC == 1 ? 4096 : 2048) + lane * 16;
  auto exchange_scores = [&](const intx16& hi, const intx16& lo) __attribute__((always_inline)) {
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
          const uint32_t at = NC == 1 ? q * 4096 + part * 1024 : q * 2048 + i * 1024;
          *(intx4*)(exchange + tile_at + at) = intx4{d[4 * i], d[4 * i + 1], d[4 * i + 2], d[4 * i + 3]};
        }
      }
    }
  };

  float sum = 0.0f, top_pt = 0.0f;
  const uint32_t lane16 = lane * 16;
  const bool lower = NC == 1 || my_block == 0;
  auto& S = ldot;  // scores
  const uint32_t first = part * kShare;  // scores i of a lane are tokens 8 (i / 4) + 4 half + i % 4, its own from here on
  const uint32_t at_max = (tb * kParts + part) * kCols + 32 * my_block + col;
  float p[kShare];
  auto store_p = [&]() __attribute__((always_inline)) {
    // Pairs in the order of bytes_to_f16; scores 8 u .. 8 u + 7 are contraction block u.
    uint8_t* to = pbuf + (tb * NC + my_block) * 2048 + lane16;
    if constexpr (NC == 1)
      *(u32x2*)(to + (part / 2) * 1024 + (part % 2) * 8) = u32x2{to_f16x2(p[0], p[2]), to_f16x2(p[1], p[3])};
    else
      *(u32x4*)(to + part * 1024) =
          u32x4{to_f16x2(p[0], p[2]), to_f16x2(p[1], p[3]), to_f16x2(p[4], p[6]), to_f16x2(p[5], p[7])};
  };
  auto weigh = [&](int i, float t, float ref, float unit) __attribute__((always_inline)) {
    const float e = __builtin_amdgcn_exp2f(__int_as_float(S[i]) - ref);
    sum += e;
    p[i] = e * t * unit;
  };
  // What a wave reads from LDS for four scores of its block: the other parts'
  // numbers, the tokens' scales.
  constexpr int kOthers = kParts - 1;
  struct SoftmaxIn {
    intx4 d[kOthers];
    floatx4 s[2];
  };
  auto read_scales = [&](uint32_t slot, int g, floatx4 (&s)[2]) __attribute__((always_inline)) {
    const float* at = (const float*)(lds + L::kAtRing + slot + L::kLat + L::kKey) + (2 * (first / 4 + g) + half) * 8;
    s[0] = *(const floatx4*)at;
    s[1] = *(const floatx4*)(at + 4);
  };
  auto read_softmax = [&](uint32_t slot, int g) __attribute__((always_inline)) {
    SoftmaxIn r;
#pragma unroll
    for (int f = 0; f < kOthers; ++f) {
      const uint32_t at = NC == 1 ? part * 4096 + ((part + 1 + f) & 3) * 1024 : part * 2048 + g * 1024;
      r.d[f] = *(const intx4*)(exchange + tile_at + at);
    }
    read_scales(slot, g, r.s);
    return r;
  };
  auto latent_scale = [](const floatx4 (&s)[2], int j) __attribute__((always_inline)) { return j < 2 ? s[0][2 * j] : s[1][2 * j - 4]; };
  auto key_token_scale = [](const floatx4 (&s)[2], int j) __attribute__((always_inline)) { return j < 2 ? s[0][2 * j + 1] : s[1][2 * j - 3]; };
  // Score i of the wave's share: its value, and what it gives with the references there are.
  auto softmax = [&](int i, const SoftmaxIn& r, float ref, float unit) __attribute__((always_inline)) {
    const int j = i % 4;
    int dot = ldot[i];
#pragma unroll
    for (int f = 0; f < kOthers; ++f) dot += r.d[f][j];
    const float t = latent_scale(r.s, j);
    S[i] = __float_as_int(fmaf((float)dot, t * lat_scale, (float)kdot[i] * (key_token_scale(r.s, j) * key_scale)));
    weigh(i, t, ref, unit);
    top_pt = fmaxf(top_pt, p[i]);
  };
  // The same of a block that some columns do not see to its end.
  auto masked = [&](uint32_t slot, uint32_t tile, float ref, float unit) __attribute__((always_inline)) {
    sum = top_pt = 0.0f;
#pragma unroll
    for (int g = 0; g < kShare / 4; ++g) {
      floatx4 s[2];
      read_scales(slot, g, s);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = 4 * g + j;
        const bool seen = tile * kLatentTile + 8 * (first / 4 + g) + 4 * half + j < limit;
        S[i] = __float_as_int(seen ? __int_as_float(S[i]) : -INFINITY);
        weigh(i, seen ? latent_scale(s, j) : 0.0f, ref, unit);  // nothing of it, not even a scale that is no number
        top_pt = fmaxf(top_pt, p[i]);
      }
    }
  };
  // Moves the references to the maxima and publishes again.
  auto move = [&](uint32_t slot, uint32_t tile) __attribute__((always_inline)) {
    float T[kShare], top = -INFINITY;  // token scales
#pragma unroll
    for (int g = 0; g < kShare / 4; ++g) {
      floatx4 s[2];
      read_scales(slot, g, s);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        T[4 * g + j] = tile * kLatentTile + 8 * (first / 4 + g) + 4 * half + j < limit ? latent_scale(s, j) : 0.0f;
        top = fmaxf(top, __int_as_float(S[4 * g + j]));
      }
    }
    auto column_max = [&](int n, float2* m) __attribute__((always_inline)) {
      *m = maxima[32 * n + col];
#pragma unroll
      for (int q = 1; q < 2 * kParts; ++q) {
        const float2 v = maxima[q * kCols + 32 * n + col];
        m->x = fmaxf(m->x, v.x), m->y = fmaxf(m->y, v.y);
      }
    };
    const float t = halves_max(top);
    if (half == 0) maxima[at_max].x = t;
    lds_barrier();
    float m[NC];
    float2 v;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      column_max(n, &v);
      m[n] = fmaxf(mref[n], v.x - 6.0f);
    }
    // log2(p * token scale) with the new ref.
    const float own = lower ? m[0] : m[NC - 1];
    float top_w = -INFINITY;
#pragma unroll
    for (int i = 0; i < kShare; ++i) top_w = fmaxf(top_w, __int_as_float(S[i]) - own + __log2f(T[i]));
    top_w = halves_max(top_w);
    if (half == 0) maxima[at_max].y = top_w;
    lds_barrier();
    if (threadIdx.x == 0) *flag = 0;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      column_max(n, &v);
      const float moved = mref[n] - m[n], w = fmaxf(fmaxf(w2[n] + moved, v.y - 6.0f), -100.0f);  // 2^-w stays a number
      const float f = __builtin_amdgcn_exp2f(moved + (w2[n] - w));
      if (NC == 1 || my_block == (uint32_t)n) l *= __builtin_amdgcn_exp2f(moved);
      mref[n] = m[n];
      w2[n] = w;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) O[i][n][j] *= f;
    }
    const float ref = lower ? mref[0] : mref[NC - 1], unit = __builtin_amdgcn_exp2f(-(lower ? w2[0] : w2[NC - 1]));
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kShare; ++i) weigh(i, T[i], ref, unit);
    store_p();
    lds_barrier();
  };
  struct KeyOperands {
    u32x4 k, hi, lo;
  };
  auto read_key = [&](uint32_t slot, int s) __attribute__((always_inline)) {
    uint32_t col = lane & 31, half = lane >> 5;
    __asm__ volatile("" : "+v"(col), "+v"(half));
    const uint32_t kk = col * kLatentRope + ((half ^ key_swizzle(col)) * 16);
    const uint8_t* kd = key_digits + my_block * 4096 + lane16 + s * 2048;
    return KeyOperands{*(const u32x4*)(lds + (L::kAtRing + L::kLat + slot + (kk ^ (32 * s)))), *(const u32x4*)kd,
                       *(const u32x4*)(kd + 1024)};
  };
  auto low = [&](int s) __attribute__((always_inline)) {
    return s < L::kLowSteps ? *(const u32x4*)(lds + L::kAtLow + s * 4096 + (wave & 3) * 1024 + lane16) : qlo[s];
  };
  auto score_codes = [&](uint32_t slot, int s) __attribute__((always_inline)) {
    return *(const u32x4*)(lds + (L::kAtRing + slot + piece(ka, part * kLatSteps + s)));
  };
  // The sums' products of the two blocks at `now`.  A step takes one operand of codes
  // and the columns' P'; its operands are read a step ahead, and no further
  // (registers).
  auto products = [&](uint32_t now, uint32_t next, const KeyOperands& key, auto move) __attribute__((always_inline)) {
    constexpr int kFrags = 4 * kBlocks;
    u32x2 codes_at[2];
    u32x4 pf[2][NC];
    auto read = [&](int f) __attribute__((always_inline)) {
      const int t = f / (2 * kBlocks), u = f / kBlocks % 2;
      codes_at[f % 2] = lds_read_tr8(lds + now + va + t * L::kTileBytes + 16 * u * RP + f % kBlocks * 256);
#pragma unroll
      for (int n = 0; n < NC; ++n)
        if (f % kBlocks == 0) pf[u][n] = *(const u32x4*)(pbuf + ((t * NC + n) * 2 + u) * 1024 + lane16);
    };
    {
      intx16 hi, lo;
      const uint32_t passed = *flag;
      const KeyOperands second = read_key(next, 1);
      score_step(key.k, key.hi, key.lo, true, hi, lo);
      score_step(second.k, second.hi, second.lo, false, hi, lo);
      read(0);
      take_keys(hi, lo);
      if (__builtin_amdgcn_readfirstlane(passed)) {
        move();
        read(0);
      }
    }
    l += sum;
#pragma unroll
    for (int f = 0; f < kFrags; ++f) {
      __builtin_amdgcn_sched_barrier(0);
      const u32x2 now_codes = codes_at[f % 2];
      if (f + 1 < kFrags) read(f + 1);
      const int i = f % kBlocks;
      if (kAll % 8 == 0 || wave + 8 * i < kAll) {
        const u32x4 v = bytes_to_f16(now_codes);
#pragma unroll
        for (int n = 0; n < NC; ++n) O[i][n] = mfma32x32x16_f16(v, pf[f / kBlocks % 2][n], O[i][n]);
      }
    }
  };

  if (threadIdx.x == 0) *flag = 0;
  latent_wait_vmcnt<0>();  // the first two blocks
  issue_two(2);
  lds_barrier();
  if (n) {
    intx16 hi, lo;
#pragma unroll
    for (int s = 0; s < kLatSteps; ++s) score_step(score_codes(tb * L::kTileBytes, s), qhi[s], low(s), s == 0, hi, lo);
    exchange_scores(hi, lo);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const KeyOperands key = read_key(tb * L::kTileBytes, s);
      score_step(key.k, key.hi, key.lo, s == 0, hi, lo);
    }
    take_keys(hi, lo);
  }
  latent_wait_vmcnt<0>();
  uint32_t now = 0, next = 2 * L::kTileBytes, free = 4 * L::kTileBytes;  // two blocks of the ring each
  for (uint32_t i = 0; i < n; i += 2) {
    lds_barrier();  // scores exchanged, the next blocks in LDS; every wave is done with the blocks before
    SoftmaxIn in = read_softmax(now + tb * L::kTileBytes, 0);
#pragma unroll
    for (int b = 0; b < 2; ++b) issue(t_begin + i + 4 + b, free + b * L::kTileBytes, i + 4 + b < n, L::kPieces);
    // The softmax, and mixed with it the latent's part of the scores of the next two
    // blocks.  Behind the last block these are of whatever the ring holds and go
    // nowhere: a second form of the loop without them took more registers than there
    // are.
    intx16 hi, lo;
    KeyOperands key;
    {
      const uint32_t tile = t_begin + i + tb;
      const bool whole = (tile + 1) * kLatentTile <= lim_min && c_last - c_first == kCols - 1;
      const float ref = lower ? mref[0] : mref[NC - 1], unit = __builtin_amdgcn_exp2f(-(lower ? w2[0] : w2[NC - 1]));
      top_pt = sum = 0.0f;
      u32x4 k = score_codes(next + tb * L::kTileBytes, 0);
      u32x4 lo_digits = low(0);
#pragma unroll
      for (int s = 0; s < kLatSteps; ++s) {
        __builtin_amdgcn_sched_barrier(0);
        const u32x4 k_now = k;
        const u32x4 lo_now = lo_digits;
        if (s + 1 < kLatSteps) k = score_codes(next + tb * L::kTileBytes, s + 1), lo_digits = low(s + 1);
        score_step(k_now, qhi[s], lo_now, s == 0, hi, lo);
        // The DMA of the two blocks behind the next two, an instruction or two a step.
#pragma unroll
        for (int d = s * 2 * L::kPieces / kLatSteps; d < (s + 1) * 2 * L::kPieces / kLatSteps; ++d) {
          const uint32_t b = d / L::kPieces, to = i + 4 + b;
          issue(t_begin + to, free + b * L::kTileBytes, to < n, d % L::kPieces);
        }
#pragma unroll
        for (int j = s * kShare / kLatSteps; j < (s + 1) * kShare / kLatSteps; ++j) {
          softmax(j, in, ref, unit);
          if (j % 4 == 3 && j + 1 < kShare) in = read_softmax(now + tb * L::kTileBytes, (j + 1) / 4);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (!whole) masked(now + tb * L::kTileBytes, tile, ref, unit);
      key = read_key(next + tb * L::kTileBytes, 0);
      store_p();
      if (fmaxf(sum, top_pt) > 16384.0f) *flag = 1;
    }
    lds_barrier();  // P' and the flag
    products(now, next + tb * L::kTileBytes, key, [&]() __attribute__((always_inline)) {
      move(now + tb * L::kTileBytes, t_begin + i + tb);
    });
    exchange_scores(hi, lo);
    latent_wait_vmcnt<0>();
    const uint32_t t = now;
    now = next, next = free, free = t;
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
// P waves take (32 columns, 8 latent elements: one store of the attention's), a
// workgroup 16 / P neighbours of them: the splits' sums weighted by 2^(m - M), a
// wave every P-th split, added in wave order, divided by the joined softmax sum and
// written as bf16 and the bf16 of what that leaves (2^-17 in all), the operands of
// the product with W_uv.  Bound by reading the partial sums: 128 splits of 128
// columns, 33 MB, 8.8 us (3.8 TB/s).
template <int RP, int NC, int P>
__global__ __launch_bounds__(1024) void latent_join_kernel(LatentAttnArgs a) {
  constexpr uint32_t kCols = 32 * NC, kPieces = 16 / P;
  __shared__ floatx4 part[16][64];
  __shared__ float2 red[16][32];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31;
  const uint32_t H = a.d.heads, cols = a.decode ? H : a.rows * H, blocks = (cols + 31) / 32;
  const uint32_t piece = blockIdx.x % (RP / 8 / kPieces) * kPieces + wave / P, block = blockIdx.x / (RP / 8 / kPieces);
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
  for (uint32_t s = wave % P; s < sq.splits; s += P) {
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
  if (wave % P != 0) return;
  float m = kNoMax;
#pragma unroll
  for (uint32_t w = 0; w < P; ++w) m = fmaxf(m, red[wave + w][col].x);
  sum = 0.0f;
  acc = floatx4{0, 0, 0, 0};
#pragma unroll
  for (uint32_t w = 0; w < P; ++w) {
    const float f = __builtin_amdgcn_exp2f(red[wave + w][col].x - m);
    sum += red[wave + w][col].y * f;
    acc += part[wave + w][lane] * f;
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
// order in LDS.  One row of 128 heads (17 MB of weights): 5.0 us.
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
  // Up to 8 splits two waves have few to go through, and idle ones would cost more:
  // one split of 6660 columns of 384 took 30 us with 16 waves of which one worked.
  uint32_t splits = 1;
  for (uint32_t b = 0; b < a.n_seqs; ++b) splits = std::max(splits, a.seqs[b].splits);
  if (splits > 8) hipLaunchKernelGGL((latent_join_kernel<RP, NC, 16>), dim3(a.blocks * (RP / 8)), dim3(1024), 0, st, a);
  else hipLaunchKernelGGL((latent_join_kernel<RP, NC, 2>), dim3(a.blocks * (RP / 64)), dim3(1024), 0, st, a);
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
