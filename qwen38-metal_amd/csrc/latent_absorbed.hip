// Latent attention, absorbed form: the queries go into the latent space
// (q_nope W_uk), attend over the 8-bit cache as over one shared key and value
// per token, and the sums of latents come out through W_uv.  For decode and
// for few rows: a token costs 584 bytes (rank 512) whatever the heads.
//
// Four launches: latent_query_kernel (which also appends the new rows),
// latent_attn_kernel (split over the cache's length), latent_join_kernel,
// latent_up_kernel.
#include <float.h>

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
// A wave takes 32 columns (heads of a row, or of several rows) and every fourth
// 32-token tile of its workgroup's share of the cache, alone: it streams the
// tiles' bytes into its own LDS ring by buffer->LDS DMA and never waits for the
// other waves before the end.
//   S^T[token][column] = codes . (hi, lo) on v_mfma_i32_32x32x32_i8, the token's
//     and the column's scales applied in fp32;
//   online softmax in fp32 (exp2 domain), p = 2^(s - ref): ref is a column's
//     maximum less 6, moved (and the sums rescaled) only when a maximum passes
//     ref + 14, so p stays below 2^14 and what is 2^-20 of the largest is still
//     a normal fp16;
//   O^T[latent element][column] += codes^T P'^T on v_mfma_f32_32x32x16_f16:
//     P' = p * token scale / 2^e, 2^e the largest scale's power of two so far,
//     rounded to fp16 (2^-11 of each term, where bf16 would be 2^-8), the codes
//     exact.
//     S^T leaves a lane the P' of its own column in the order that the second
//     product wants once the tokens of its operand are taken in the same order,
//     so P' stays in registers; the codes' operand comes by transposing reads.
// The O^T accumulators (rank_pad x 32 fp32) take half of the register file.
template <int RP>
struct AbsorbedLds {
  static constexpr int kChunks = RP / 16;  // 16-byte pieces of a latent
  static constexpr int kLat = kLatentTile * RP, kKey = kLatentTile * (int)kLatentRope, kScale = kLatentTile * 8;
  static constexpr int kTileBytes = kLat + kKey + kScale;
  static constexpr int kRing = RP >= 384 ? 2 : RP == 256 ? 3 : 4;
  static constexpr int kPad = 132;  // floats of a column's 128 sums in the final merge
  static constexpr int kMerge = 4 * (int)kLatentCols * kPad * 4 + 4 * (int)kLatentCols * 8;
  static constexpr int kBytes = 4 * kRing * kTileBytes > kMerge ? 4 * kRing * kTileBytes : kMerge;
  static constexpr int kDma = RP / 32 + 3;  // DMA instructions of a tile
};

// Order of a token's 16-byte pieces in LDS: piece j at j ^ swizzle(token).  Both
// the reads of one piece of 8 consecutive tokens and those of the 8 tokens of a
// transposing read (0..3, 8..11 or 4..7, 12..15) fall on different banks.
__device__ __forceinline__ constexpr uint32_t lat_swizzle(uint32_t tok) {
  return (tok & 3) | ((((tok >> 2) ^ (tok >> 3)) & 1) << 2);
}

template <int RP>
__global__ __launch_bounds__(256, 1) void latent_attn_kernel(LatentAttnArgs a) {
  using L = AbsorbedLds<RP>;
  constexpr int CH = L::kChunks, kLatSteps = RP / 32, kBlocks = RP / 32;
  constexpr uint32_t kStride = RP + kLatentRope;
  __shared__ __attribute__((aligned(16))) uint8_t lds[L::kBytes];
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t col = lane & 31, half = lane >> 5;
  const uint32_t unit = blockIdx.x, H = a.d.heads;
  uint32_t b = 0;
  while (b + 1 < a.n_seqs && unit >= a.seqs[b + 1].unit_begin) ++b;
  const LatentSeq& sq = a.seqs[b];
  const uint32_t cols = a.decode ? H : a.rows * H;
  const uint32_t blocks = (cols + kLatentCols - 1) / kLatentCols;
  const uint32_t local = unit - sq.unit_begin, cb = local % blocks, split = local / blocks;
  // Tokens that a column sees: up to its own row.
  const uint32_t c_first = cb * kLatentCols, c_last = min(c_first + kLatentCols, cols) - 1, c = c_first + col;
  const uint32_t lim_min = sq.start + c_first / H + 1, lim_max = sq.start + c_last / H + 1;
  const uint32_t limit = c <= c_last ? sq.start + c / H + 1 : 0;
  const uint32_t tiles = (lim_max + kLatentTile - 1) / kLatentTile;
  const uint32_t t_begin = split * a.tiles_per_split, t_end = min(tiles, t_begin + a.tiles_per_split);

  const size_t block = sq.block_begin + cb;
  u32x4 qhi[kLatSteps + 2], qlo[kLatSteps + 2];
  {
    const uint8_t* dg = a.digits + block * latent_digit_bytes(RP) + lane * 32;
#pragma unroll
    for (int s = 0; s < kLatSteps + 2; ++s) {
      qhi[s] = *(const u32x4*)(dg + s * 2048);
      qlo[s] = *(const u32x4*)(dg + s * 2048 + 16);
    }
  }
  const float2 qs = limit ? *(const float2*)(a.qscale + (block * kLatentCols + col) * 2) : float2{0.0f, 0.0f};
  const float lat_scale = qs.x * a.scale * kLog2e, key_scale = qs.y * a.scale * kLog2e;

  uint8_t* ring = lds + wave * (L::kRing * L::kTileBytes);
  const uint32_t tpi = 64 / CH;  // tokens of a DMA instruction (a whole number but for rank_pad 384)
  const uint32_t jb = lane % CH, tb = lane / CH;
  const uint32_t j16 = (jb ^ lat_swizzle(tb)) * 16, tb_off = tb * kStride;
  const uint32_t key_tok = lane / 4;
  auto issue = [&](uint32_t tile, uint32_t slot) __attribute__((always_inline)) {
    uint8_t* to = ring + slot * L::kTileBytes;
    const auto rows = latent_rsrc(sq.rows.codes + (size_t)tile * kLatentTile * kStride, kLatentTile * kStride);
#pragma unroll
    for (int i = 0; i < RP / 32; ++i) {
      if constexpr (64 % CH == 0) {
        latent_dma16(rows, to + i * 1024, tb_off + (j16 ^ (lat_swizzle(i * tpi) * 16)), i * tpi * kStride);
      } else {
        const uint32_t p = i * 64 + lane, tok = p / CH, j = (p % CH) ^ lat_swizzle(tok);
        latent_dma16(rows, to + i * 1024, tok * kStride + j * 16, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)  // token i * 16 + lane / 4, piece (lane % 4) ^ (token / 2 % 4)
      latent_dma16(rows, to + L::kLat + i * 1024,
                   (i * 16 + key_tok) * kStride + RP + (((lane & 3) ^ ((key_tok >> 1) & 3)) * 16), 0);
    const auto scales = latent_rsrc(sq.rows.scales + (size_t)tile * kLatentTile * 2, kLatentTile * 8);
    latent_dma4(scales, to + L::kLat + L::kKey, lane * 4);
  };

  // LDS offsets of this lane: codes of token `col` (score operand) and of the 8
  // tokens of a transposing read.
  const uint32_t sw = lat_swizzle(col);
  uint32_t ka[4], va[4];
  const uint32_t trow = (lane & 15) >> 1, vtok = 4 * half + (trow < 4 ? trow : trow + 4);
#pragma unroll
  for (uint32_t v = 0; v < 4; ++v) {
    ka[v] = col * RP + (((2 * v + half) ^ sw) * 16);
    va[v] = vtok * RP + (((2 * v + ((lane >> 4) & 1)) ^ lat_swizzle(vtok)) * 16) + 8 * (lane & 1);
  }

  floatx16 O[kBlocks];
#pragma unroll
  for (int i = 0; i < kBlocks; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) O[i][j] = 0.0f;
  float mref = kNoMax, l = 0.0f;
  uint32_t vexp = 0x00800000u;  // the largest token scale's exponent, as a float's bits: the sums' unit

  const uint32_t first = t_begin + wave;
  const uint32_t count = first < t_end ? (t_end - first + 3) / 4 : 0;
#pragma unroll
  for (int i = 0; i < L::kRing - 1; ++i)
    if ((uint32_t)i < count) issue(first + 4 * i, i);
  uint32_t slot = 0;
  for (uint32_t it = 0; it < count; ++it) {
    const uint32_t tile = first + 4 * it;
    if (it + L::kRing - 1 < count) {
      const uint32_t to = slot + L::kRing - 1;
      issue(tile + 4 * (L::kRing - 1), to >= L::kRing ? to - L::kRing : to);
      latent_wait_vmcnt<L::kDma*(L::kRing - 1) < 63 ? L::kDma * (L::kRing - 1) : 63>();
    } else {
      latent_wait_vmcnt<0>();
    }
    const uint8_t* lat = ring + slot * L::kTileBytes;
    const uint8_t* key = lat + L::kLat;
    const float* scales = (const float*)(key + L::kKey);

    // Scores: the shared key's part, then the latent's.  A step's operand is read
    // two steps ahead; the compiler barriers keep that order, and keep the reads
    // from running further ahead (the columns' queries and the sums leave about a
    // hundred registers).
    float S[16];
    auto key_at = [&](int s) __attribute__((always_inline)) {
      return s < 2 ? *(const u32x4*)(key + col * kLatentRope + (((2 * s + half) ^ ((col >> 1) & 3)) * 16))
                   : *(const u32x4*)(lat + ka[(s - 2) & 3] + ((s - 2) >> 2) * 128);
    };
    {
      constexpr int kAhead = 2;
      u32x4 kf[kAhead + 1];
#pragma unroll
      for (int s = 0; s < kAhead; ++s) kf[s] = key_at(s);
      intx16 hi = {}, lo = {};
#pragma unroll
      for (int s = 0; s < kLatSteps + 2; ++s) {
        if (s + kAhead < kLatSteps + 2) kf[(s + kAhead) % (kAhead + 1)] = key_at(s + kAhead);
        __asm__ volatile("" ::: "memory");
        const int qi = s < 2 ? kLatSteps + s : s - 2;
        hi = mfma32x32x32_i8(kf[s % (kAhead + 1)], qhi[qi], hi);
        lo = mfma32x32x32_i8(kf[s % (kAhead + 1)], qlo[qi], lo);
        if (s == 1) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float ks = scales[(8 * (i / 4) + 4 * half + i % 4) * 2 + 1];
            S[i] = (float)((hi[i] << 8) + lo[i]) * (ks * key_scale);
            hi[i] = lo[i] = 0;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float ls = scales[(8 * (i / 4) + 4 * half + i % 4) * 2];
        // (At most 512 * 127 * 127 * 256 + 512 * 128 * 127 < 2^31.)
        S[i] = fmaf((float)((hi[i] << 8) + lo[i]), ls * lat_scale, S[i]);
      }
    }
    // A tile's largest token scale, as a power of two: P' is kept relative to the
    // largest so far.
    const uint32_t tok0 = tile * kLatentTile + 4 * half;
    const bool whole = (tile + 1) * kLatentTile <= lim_min && c_last - c_first == kLatentCols - 1;
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 16; ++i) S[i] = tok0 + 8 * (i / 4) + i % 4 < limit ? S[i] : -INFINITY;
    }
    // Not of tokens behind the block's last, whose scales are any bits, nor NaN.
    const float own = tile * kLatentTile + col < lim_max && scales[2 * col] <= FLT_MAX ? scales[2 * col] : 0.0f;
    const uint32_t big = __float_as_uint(wave_allmax(own)) & 0x7F800000u;
    float top = S[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, S[i]);
    top = halves_max(top);
    if (__any(top > mref + 14.0f) || big > vexp) {
      const float m = fmaxf(mref, top - 6.0f);
      const uint32_t e = max(big, vexp);
      float f = __builtin_amdgcn_exp2f(mref - m);
      mref = m;
      l *= f;
      f *= __uint_as_float(max((int)(vexp - e + 0x3F800000u), 0));  // 2^(old - new)
      vexp = e;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) O[i][j] *= f;
    }
    const float unit_scale = __uint_as_float(0x7F000000u - vexp);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      S[i] = __builtin_amdgcn_exp2f(S[i] - mref);
      l += S[i];
      const float ls = scales[(8 * (i / 4) + 4 * half + i % 4) * 2];
      S[i] *= (whole || tok0 + 8 * (i / 4) + i % 4 < limit ? ls : 0.0f) * unit_scale;
    }
    u32x4 p[2];  // pairs in the order of bytes_to_f16
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        p[u][2 * i] = to_f16x2(S[8 * u + 4 * i], S[8 * u + 4 * i + 2]);
        p[u][2 * i + 1] = to_f16x2(S[8 * u + 4 * i + 1], S[8 * u + 4 * i + 3]);
      }
    {
      constexpr int kAhead = 4;
      u32x2 vf[kAhead + 1];
      auto value_at = [&](int i) __attribute__((always_inline)) {
        return lds_read_tr8(lat + va[i / 2 & 3] + (i / 8) * 128 + (i & 1) * 16 * RP);
      };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) vf[i] = value_at(i);
#pragma unroll
      for (int i = 0; i < 2 * kBlocks; ++i) {
        if (i + kAhead < 2 * kBlocks) vf[(i + kAhead) % (kAhead + 1)] = value_at(i + kAhead);
        __asm__ volatile("" ::: "memory");
        O[i / 2] = mfma32x32x16_f16(bytes_to_f16(vf[i % (kAhead + 1)]), p[i & 1], O[i / 2]);
      }
    }
    latent_wait_lds();  // before the DMA of a later tile writes here
    slot = slot + 1 == L::kRing ? 0 : slot + 1;
  }

  // Merge the four waves: one maximum per column, then the sums, 128 latent
  // elements at a time.
  l = halves_sum(l);
  __syncthreads();
  float* ml = (float*)(lds + 4 * kLatentCols * L::kPad * 4);
  if (half == 0) *(float2*)(ml + (wave * kLatentCols + col) * 2) = float2{mref, l};
  __syncthreads();
  float m = kNoMax, sum = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[(w * kLatentCols + col) * 2]);
#pragma unroll
  for (int w = 0; w < 4; ++w)
    sum += ml[(w * kLatentCols + col) * 2 + 1] * __builtin_amdgcn_exp2f(ml[(w * kLatentCols + col) * 2] - m);
  const float f = __builtin_amdgcn_exp2f(mref - m) * __uint_as_float(vexp);
  if (wave == 0 && half == 0)
    *(float2*)(a.partials + (size_t)a.units * kLatentCols * RP + ((size_t)unit * kLatentCols + col) * 2) =
        float2{m, sum};
  float* buf = (float*)lds;
#pragma unroll
  for (int q = 0; q < RP / 128; ++q) {
#pragma unroll
    for (int rb = 0; rb < 4; ++rb)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        floatx4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = O[4 * q + rb][4 * g + i] * f;
        *(floatx4*)(buf + (wave * kLatentCols + col) * L::kPad + 32 * rb + 8 * g + 4 * half) = v;
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = i * 256 + threadIdx.x, cc = at / 32, r = (at % 32) * 4;
      if (c_first + cc > c_last) break;
      floatx4 v = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < 4; ++w) v += *(const floatx4*)(buf + (w * kLatentCols + cc) * L::kPad + r);
      *(floatx4*)(a.partials + ((size_t)unit * kLatentCols + cc) * RP + q * 128 + r) = v;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Joining the splits, and out of the latent space
// ---------------------------------------------------------------------------
// Workgroup = (one (row, head) column, 128 latent elements): its splits' sums
// weighted by 2^(m - M), eight splits at a time, divided by the joined softmax
// sum and written as bf16 and the bf16 of what that leaves (2^-17 in all), the
// operands of the product with W_uv.
template <int RP>
__global__ __launch_bounds__(256) void latent_join_kernel(LatentAttnArgs a) {
  __shared__ floatx4 part[256];
  const uint32_t c_all = blockIdx.x / (RP / 128), r0 = blockIdx.x % (RP / 128) * 128;
  const uint32_t H = a.d.heads, m = c_all / H, h = c_all - m * H;
  const LatentSeq& sq = a.seqs[a.decode ? m : 0];
  const uint32_t cols = a.decode ? H : a.rows * H, blocks = (cols + kLatentCols - 1) / kLatentCols;
  const uint32_t c = a.decode ? h : c_all, cb = c / kLatentCols, col = c % kLatentCols;
  const uint32_t t = threadIdx.x % 32, group = threadIdx.x / 32, lane = threadIdx.x & 63;
  const float* ml = a.partials + (size_t)a.units * kLatentCols * RP;
  auto at = [&](uint32_t s) { return (size_t)(sq.unit_begin + s * blocks + cb) * kLatentCols + col; };
  float top = kNoMax, sum = 0.0f;
  for (uint32_t s = lane; s < sq.splits; s += 64) top = fmaxf(top, ml[at(s) * 2]);
  top = wave_allmax(top);
  for (uint32_t s = lane; s < sq.splits; s += 64) {
    const float2 v = *(const float2*)(ml + at(s) * 2);
    sum += v.y * __builtin_amdgcn_exp2f(v.x - top);
  }
  sum = wave_allsum(sum);
  floatx4 acc = {0, 0, 0, 0};
#pragma unroll 4
  for (uint32_t s = group; s < sq.splits; s += 8) {
    const float w = __builtin_amdgcn_exp2f(ml[at(s) * 2] - top);
    acc += *(const floatx4*)(a.partials + at(s) * RP + r0 + 4 * t) * w;
  }
  part[threadIdx.x] = acc;
  __syncthreads();
  if (group != 0) return;
#pragma unroll
  for (int g = 1; g < 8; ++g) acc += part[g * 32 + t];
  const float r = 1.0f / sum;
  float x[4], y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = acc[i] * r;
    y[i] = x[i] - (float)(__bf16)x[i];
  }
  uint16_t* to = a.mixed + (size_t)c_all * 2 * RP + r0 + 4 * t;
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

template <int RP>
hipError_t absorbed(const LatentAttnArgs& a, hipStream_t st) {
  const uint32_t tiles = (a.rows + 15) / 16 * a.d.heads, append_blocks = (a.rows + 3) / 4;
  hipLaunchKernelGGL(latent_query_kernel<RP>, dim3(append_blocks + tiles * (RP / 128)), dim3(256), 0, st, a, append_blocks);
  hipLaunchKernelGGL(latent_attn_kernel<RP>, dim3(a.units), dim3(256), 0, st, a);
  hipLaunchKernelGGL(latent_join_kernel<RP>, dim3(a.rows * a.d.heads * (RP / 128)), dim3(256), 0, st, a);
  hipLaunchKernelGGL(latent_up_kernel<RP>, dim3(tiles * (a.d.v_pad / 32)), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_latent_absorbed(const LatentAttnArgs& a, hipStream_t st) {
  switch (a.d.rank_pad) {
    case 128: return absorbed<128>(a, st);
    case 256: return absorbed<256>(a, st);
    case 384: return absorbed<384>(a, st);
    default: return absorbed<512>(a, st);
  }
}

}  // namespace qm
