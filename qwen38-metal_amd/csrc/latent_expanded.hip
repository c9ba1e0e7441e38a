// Latent attention, expanded form: keys and values of every head are formed
// from the cached latents, once for all rows of the call, and the rows attend
// over them.  For prompts: with many rows a (row, token) pair costs nope + rope
// + v multiplications a head where the absorbed form needs 2 rank + rope.
//
// Three launches, the last two for as many heads at a time as the workspace
// holds: latent_unpack_kernel, latent_expand_kernel (the GEMM), and
// latent_prompt_kernel.
//
// Everything between them lies in global memory in operand order: a block of 32
// rows (tokens, or weight rows) x 16 contraction elements is 1 KB in which lane
// l's 16 bytes are row l % 32, elements 8 (l / 32) .. + 7 (or, where the
// elements come out of an MFMA, the eight that one lane holds: see expand).
// Loads, LDS and stores are then linear: whole cache lines, no bank conflicts.
//
// Keys and values are fp16 (2^-11 of each; bf16 would be 2^-8), kept in its
// range by powers of two: the weights' per head (wmul: 127 sum |W| of a row stays
// below 2^15), the tokens' per tile of 32 (2^g: the largest scale is below 1),
// and each query row's.  The powers come back exactly in fp32.  Under a tile's
// power the values of a token whose latent scale is more than 2^19 below the largest
// of its 32 lose bits; so does a part of a score (nope, rope) that is 2^20 below the
// other in the query and above it in the token.
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "latent.h"
#include "latent_device.h"

namespace qm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoMax = -1e30f;
constexpr int kKeyPower = 8;

// ---------------------------------------------------------------------------
// Weights
// ---------------------------------------------------------------------------
// wmul[h] = {W_uk's power of two, W_uv's}: 127 * (largest row sum of |W|) * wmul
// in [2^14, 2^15), or up to a quarter of that where the sum times 127 would pass fp32.  Rows with
// a number that is none have no say: what they give is none at any power, and the
// head's other values keep their bits.
__global__ __launch_bounds__(256) void latent_wmul_kernel(LatentDims d, const uint16_t* up, float* wmul) {
  __shared__ float top[2][4];
  const uint32_t h = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rows = d.nope_pad + d.v_pad;
  float best[2] = {0.0f, 0.0f};
#pragma unroll 4
  for (uint32_t n = wave; n < rows; n += 4) {
    const uint16_t* w = up + ((size_t)h * rows + n) * d.rank_pad;
    const u32x4 x = 8 * lane < d.rank_pad ? *(const u32x4*)(w + 8 * lane) : u32x4{0, 0, 0, 0};
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) s += fabsf(bf16_to_f32(x[k] & 0xFFFFu)) + fabsf(__uint_as_float(x[k] & 0xFFFF0000u));
    s = wave_allsum(s);
    const int part = n >= d.nope_pad;
    best[part] = fmaxf(best[part], s <= FLT_MAX ? s : 0.0f);
  }
  if (lane == 0) top[0][wave] = best[0], top[1][wave] = best[1];
  __syncthreads();
  if (threadIdx.x < 2) {
    float s = 0.0f;
    for (int w = 0; w < 4; ++w) s = fmaxf(s, top[threadIdx.x][w]);
    int e = 0;
    // (Rows of nothing: any power will do.)
    if (s > 0.0f) e = s <= FLT_MAX / 127.0f ? 14 - ilogbf(s * 127.0f) : 7 - ilogbf(s);
    wmul[2 * h + threadIdx.x] = ldexpf(1.0f, std::min(std::max(e, -120), 120));
  }
}

// wop: fp16 W * wmul in operand order, [H * rows / 32][rank_pad / 16][64 lanes][8].
__global__ __launch_bounds__(256) void latent_wop_kernel(LatentDims d, const uint16_t* up, const float* wmul,
                                                         uint16_t* wop) {
  const uint32_t rows = d.nope_pad + d.v_pad, steps = d.rank_pad / 16;
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;  // one lane's 16 bytes
  const uint32_t lane = i & 63, step = (uint32_t)((i >> 6) % steps);
  const size_t n = (i >> 6) / steps * 32 + lane % 32;
  if (n >= (size_t)d.heads * rows) return;
  const uint32_t h = (uint32_t)(n / rows);
  const float mul = wmul[2 * h + (n % rows >= d.nope_pad)];
  const u32x4 w = *(const u32x4*)(up + n * d.rank_pad + 16 * step + 8 * (lane / 32));
  u32x4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    v[k] = to_f16x2(bf16_to_f32(w[k] & 0xFFFFu) * mul, __uint_as_float(w[k] & 0xFFFF0000u) * mul);
  *(u32x4*)(wop + 8 * i) = v;
}

// ---------------------------------------------------------------------------
// Latents and shared keys out of the cache
// ---------------------------------------------------------------------------
// A workgroup takes a tile of 32 tokens: codes to fp16 (exact) in operand order;
// the shared key scaled, likewise; the tokens' factors.  Tokens behind the last
// become zeros.
//   g = 1 + exponent of the tile's largest scale (latent or key), gv of its
//   largest latent scale; key operand 2^8 code * s_key / 2^g (kKeyPower: below 2^15,
//   as the expanded keys are), fk = s_lat / 2^g, fv = s_lat / 2^gv, powers = {2^g,
//   2^gv}.
// A token that stands for NaN keeps it in its key (fk or the operand) and has fv
// = 0: rows that do not see it multiply its value by 0.
// 6144 tokens of 512 + 64 (3.6 MB in, 7.2 MB out): 9.0 us; 1024: 5.8, a launch and a
// chain of two loads.
__global__ __launch_bounds__(256) void latent_unpack_kernel(LatentExpandArgs a) {
  __shared__ float sl[32], sk[32];
  const uint32_t tile = blockIdx.x, tid = threadIdx.x, rp = a.d.rank_pad, stride = rp + kLatentRope;
  const uint32_t lane = tid & 63, tok = tile * 32 + lane % 32;
  const bool live = tok < a.tokens;
  if (tid < 64) {
    float2 s = live ? *(const float2*)(a.rows.scales + 2 * (size_t)tok) : float2{0.0f, 0.0f};
    float top = fmaxf(s.x <= FLT_MAX ? s.x : 0.0f, s.y <= FLT_MAX ? s.y : 0.0f);
    float topv = s.x <= FLT_MAX ? s.x : 0.0f;
    top = wave_allmax(top), topv = wave_allmax(topv);
    // 2^g as a float's bits: the exponent field, plus one (at most 2^122: scales
    // end at FLT_MAX / 127).  Both are kept from vanishing: 2^g is in the scores'
    // factor, the softmax sum is over 2^gv.
    const uint32_t g = max(__float_as_uint(top) & 0x7F800000u, 0x21800000u) + 0x00800000u;
    const uint32_t gv = max(__float_as_uint(topv) & 0x7F800000u, 0x21800000u) + 0x00800000u;
    const float ig = __uint_as_float(0x7F000000u - g), igv = __uint_as_float(0x7F000000u - gv);
    if (lane < 32) {
      sk[lane] = s.y * ig * (float)(1 << kKeyPower);
      a.fk[tok] = s.x * ig;
      a.fv[tok] = s.x <= FLT_MAX ? s.x * igv : 0.0f;
    }
    if (lane == 0) *(float2*)(a.powers + 2 * tile) = float2{__uint_as_float(g), __uint_as_float(gv)};
  }
  __syncthreads();
  const int8_t* row = a.rows.codes + (size_t)(live ? tok : 0) * stride + 8 * (lane / 32);
  for (uint32_t s = tid >> 6; s < rp / 16 + 4; s += 4) {  // a wave takes a 1 KB block
    const u32x2 c = live ? *(const u32x2*)(row + 16 * s) : u32x2{0, 0};
    const bool key = s >= rp / 16;
    const float f = key ? sk[lane % 32] : 1.0f;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)(int8_t)(c[i / 4] >> (8 * (i % 4))) * f;
    const u32x4 v = {to_f16x2(x[0], x[1]), to_f16x2(x[2], x[3]), to_f16x2(x[4], x[5]), to_f16x2(x[6], x[7])};
    uint16_t* to = key ? a.keys + ((size_t)tile * 4 + s - rp / 16) * 512 : a.latents + ((size_t)tile * (rp / 16) + s) * 512;
    *(u32x4*)(to + 8 * lane) = v;
  }
}

// ---------------------------------------------------------------------------
// Keys and values
// ---------------------------------------------------------------------------
// Workgroup = 128 tokens x 256 weight rows, a wave 128 x 64 of them (all keys or
// all values: the parts of a head are multiples of 64).  Both operands stream
// through LDS, 32 contraction elements a stage, by buffer->LDS DMA.
//   Keys: D = W (rows) x latents (columns): a lane holds, for its token, the key
//   elements 16 u + 4 h + {0..3}, + 8 + {0..3} (h = lane / 32) in eight registers:
//   the 16 bytes of contraction block u of the prompt kernel's key operand, whose
//   queries are read in the same order.
//   Values: D = latents (rows) x W (columns): a lane holds, for its value
//   element, the tokens in the order in which the prompt kernel's weights P lie.
// Bound by the loop of a stage (barrier, LDS reads of 12 KB a wave, 16 products):
// 6144 tokens x 32768 rows x 512 take 240 us, 860 TFLOP/s, the matrix cores 44% busy
// at two workgroups a CU; 393 MB are written meanwhile, without which a like loop
// took a tenth less.
constexpr int kExpRows = 256, kExpTokens = 128, kExpStages = 3;
constexpr int kExpStageBytes = (kExpTokens + kExpRows) * 64;

template <int RP>
__global__ __launch_bounds__(256, 2) void latent_expand_kernel(LatentExpandArgs a) {
  constexpr int kSteps = RP / 32;  // stages
  __shared__ __attribute__((aligned(16))) uint8_t lds[kExpStages * kExpStageBytes];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t rows = a.d.nope_pad + a.d.v_pad, total = a.heads * rows;
  const uint32_t t_tiles = a.padded / kExpTokens;
  const uint32_t tb = blockIdx.x % t_tiles, nb = blockIdx.x / t_tiles;
  const uint32_t n_first = nb * kExpRows;                   // row among the chunk's
  const uint32_t n_blocks = min(kExpRows, total - n_first) / 32;
  const uint8_t* lat = (const uint8_t*)a.latents + (size_t)tb * 4 * (RP / 16) * 1024;
  const uint8_t* wop = (const uint8_t*)a.wop + ((size_t)a.head0 * rows + n_first) / 32 * (RP / 16) * 1024;
  const auto ra = latent_rsrc(lat, 4 * (RP / 16) * 1024);
  const auto rw = latent_rsrc(wop, n_blocks * (RP / 16) * 1024);
  // A stage's 24 KB: 4 token blocks, then 8 row blocks, 2 KB (two contraction
  // blocks) each; wave w brings every fourth KB.  Behind the last row block comes
  // it again, for waves that store nothing.
  auto issue = [&](int s, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 6; ++i) {
      const uint32_t kb = 4 * i + wave, blk = kb / 2, u = kb & 1;
      uint8_t* to = lds + buf * kExpStageBytes + kb * 1024;
      if (i < 2) latent_dma16(ra, to, lane * 16, (blk * (RP / 16) + 2 * s + u) * 1024);
      else latent_dma16(rw, to, lane * 16, (min(blk - 4, n_blocks - 1) * (RP / 16) + 2 * s + u) * 1024);
    }
  };
  floatx16 acc[4][2];  // [token block][row block]
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[t][n][i] = 0.0f;
  const uint32_t n0 = n_first + 64 * wave, head = n0 / rows, in_head = n0 - head * rows;
  const bool keys = in_head < a.d.nope_pad;
  auto stage = [&](int buf, auto key_part) __attribute__((always_inline)) {
    const uint8_t* A = lds + buf * kExpStageBytes + lane * 16;
    const uint8_t* B = A + 8192 + wave * 4096;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      u32x4 x[4], w[2];
#pragma unroll
      for (int t = 0; t < 4; ++t) x[t] = *(const u32x4*)(A + t * 2048 + u * 1024);
#pragma unroll
      for (int n = 0; n < 2; ++n) w[n] = *(const u32x4*)(B + n * 2048 + u * 1024);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int n = 0; n < 2; ++n)
          acc[t][n] = decltype(key_part)::value ? mfma32x32x16_f16(w[n], x[t], acc[t][n])
                                                : mfma32x32x16_f16(x[t], w[n], acc[t][n]);
    }
  };
  issue(0, 0);
  issue(1, 1);
  auto walk = [&](auto key_part) __attribute__((always_inline)) {
    int buf = 0;
    for (int s = 0; s < kSteps; ++s) {
      if (s + 1 < kSteps) latent_wait_vmcnt<6>();
      else latent_wait_vmcnt<0>();
      lds_barrier();  // stage s is in LDS; every wave is done with stage s - 1
      if (s + 2 < kSteps) issue(s + 2, buf == 0 ? 2 : buf - 1);
      stage(buf, key_part);
      buf = buf == 2 ? 0 : buf + 1;
    }
  };
  if (keys) walk(std::true_type{});
  else walk(std::false_type{});
  if (n0 >= total) return;
  const uint32_t tile0 = tb * 4;
  if (keys) {
    // [head][tile][nope_pad / 16][64][8]
    const uint32_t steps = a.d.nope_pad / 16;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const float f = a.fk[(tile0 + t) * 32 + lane % 32];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          u32x4 v;
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = to_f16x2(acc[t][n][8 * u + 2 * i] * f, acc[t][n][8 * u + 2 * i + 1] * f);
          *(u32x4*)(a.k + (((size_t)head * (a.padded / 32) + tile0 + t) * steps + in_head / 16 + 2 * n + u) * 512 +
                    8 * lane) = v;
        }
    }
  } else {
    // [head][tile][v_pad / 32][2][64][8]
    const uint32_t blocks = a.d.v_pad / 32;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      float f[16];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const floatx4 x = *(const floatx4*)(a.fv + (tile0 + t) * 32 + 8 * g + 4 * (lane / 32));
#pragma unroll
        for (int i = 0; i < 4; ++i) f[4 * g + i] = x[i];
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          u32x4 v;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[i] = to_f16x2(acc[t][n][8 * u + 2 * i] * f[8 * u + 2 * i],
                            acc[t][n][8 * u + 2 * i + 1] * f[8 * u + 2 * i + 1]);
          *(u32x4*)(a.v + ((((size_t)head * (a.padded / 32) + tile0 + t) * blocks + (in_head - a.d.nope_pad) / 32 + n) * 2 +
                           u) * 512 + 8 * lane) = v;
        }
    }
  }
}

// ---------------------------------------------------------------------------
// Attention over expanded keys and values
// ---------------------------------------------------------------------------
// Workgroup = (32 W rows, head), wave = 32 rows, the rows as MFMA columns:
//   S^T[token][row] = K Q^T, online softmax in fp32 with a lane's column to
//   itself, O^T[v][row] += V^T P^T with P (fp16) straight from the registers that
//   held S.  Tiles of 32 tokens stream through LDS by DMA, shared by the waves.
// P = 2^(s + gv - ref), 2^gv the tile's power of two of the values and ref the
// row's maximum of s + gv less 6; the softmax sum takes a tile's sum of P over
// 2^gv.  A tile is weighed with the ref there is; only where a lane's sum of P
// passes 2^14 (so that no P can have passed fp16) is its maximum looked for, ref
// moved, the sums rescaled and the tile weighed again.
//
// Bound by the matrix cores and the vector unit together (640 and 480 cycles a wave
// and tile, two waves a SIMD): 2048 rows of 128 heads on 4096 tokens take about 900
// us (853 at the least), 58% of the matrix cores' cycles.  The next tile's key
// products go between the exponentials; with each phase by itself, and a maximum
// for every tile: 7% more.  1024 rows of 64 heads take 38 to 40 us, 6 of them until
// the queries (25 MB, all at once) are there.
template <int NP, int VP, int W>
struct PromptLds {
  static constexpr int kKSteps = NP / 16 + 4, kVBlocks = VP / 32;
  static constexpr int kTile = (kKSteps + 2 * kVBlocks) * 1024;
  static constexpr int kTiles = 2;  // of a stage
  static constexpr int kBufs = 3;
  static constexpr int kStage = kTiles * kTile;
  static constexpr int kDma = kStage / 1024 / W;  // DMA instructions of a wave
  static_assert(kDma * W * 1024 == kStage, "every wave brings as much");
};

template <int NP, int VP, int W>
__global__ __launch_bounds__(64 * W, 2) void latent_prompt_kernel(LatentExpandArgs a) {
  using L = PromptLds<NP, VP, W>;
  constexpr int KS = L::kKSteps, VB = L::kVBlocks;
  __shared__ __attribute__((aligned(16))) uint8_t lds[L::kBufs * L::kStage];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t col = lane & 31, half = lane >> 5;
  const uint32_t hc = blockIdx.x % a.heads, rb = gridDim.x / a.heads - 1 - blockIdx.x / a.heads;
  const uint32_t h = a.head0 + hc, H = a.d.heads, nope = a.d.nope, qw = nope + a.d.rope;
  // Paired: 128 rows from the end for waves 0..3, as many from the start for 4..7 (of
  // an odd number of such blocks the middle one has a workgroup's first waves alone).
  const uint32_t halves = (a.m + 127) / 128, last = halves - 1 - rb;
  const bool none = a.paired && wave >= 4 && rb == last;
  const uint32_t r0 = none ? a.m : !a.paired ? (rb * W + wave) * 32 : (wave < 4 ? last : rb) * 128 + wave % 4 * 32;
  const uint32_t r_end = a.paired ? (last + 1) * 128 : (rb + 1) * 32 * W, row = r0 + col;
  const bool live = row < a.m;
  // Tokens that the workgroup, the wave and the lane see.
  const uint32_t wg_limit = a.start + min(r_end, a.m);
  const uint32_t wave_limit = r0 < a.m ? a.start + min(r0 + 32, a.m) : 0;
  const uint32_t wave_whole = r0 < a.m ? a.start + r0 + 1 : 0;  // every row sees what is below
  const uint32_t limit = live ? a.start + row + 1 : 0;

  const uint32_t tiles = (wg_limit + 31) / 32, stages = (tiles + L::kTiles - 1) / L::kTiles;
  const uint32_t all_tiles = a.padded / 32;
  const uint8_t* kb = (const uint8_t*)a.k + (size_t)hc * all_tiles * (NP / 16) * 1024;
  const uint8_t* vb = (const uint8_t*)a.v + (size_t)hc * all_tiles * (2 * VB) * 1024;
  const uint8_t* sb = (const uint8_t*)a.keys;
  // What this wave copies of a stage: addresses in the next stage to issue.
  const uint8_t* from[L::kDma];
  uint32_t step[L::kDma];
#pragma unroll
  for (int i = 0; i < L::kDma; ++i) {
    const uint32_t kbyte = i * W + wave, t = kbyte / (L::kTile / 1024), at = kbyte - t * (L::kTile / 1024);
    const uint32_t per = at < NP / 16 ? NP / 16 : at < KS ? 4 : 2 * VB;
    const uint8_t* part = at < NP / 16 ? kb + at * 1024 : at < KS ? sb + (at - NP / 16) * 1024 : vb + (at - KS) * 1024;
    from[i] = part + (size_t)t * per * 1024;
    step[i] = L::kTiles * per * 1024;
  }
  auto issue = [&](uint32_t buf) __attribute__((always_inline)) {  // within the padding: padded is a multiple of 128
#pragma unroll
    for (int i = 0; i < L::kDma; ++i) {
      latent_dma16(latent_rsrc(from[i], 1024), lds + buf * L::kStage + (i * W + wave) * 1024, lane * 16, 0);
      from[i] += step[i];
    }
  };
  issue(0);
  if (stages > 1) issue(1);

  // Queries, in the key operand's order: fp16 times 2^f, the expanded part divided
  // by the weights' power as well and the shared one by the key operand's, f the
  // largest that keeps both parts below 2^15.  With keys as large, the smaller part
  // of a query and the smaller of a token may be 2^20 below the larger ones before
  // fp16 holds them in fewer than 11 bits.  The scale goes in with its mantissa, so that products become exponents
  // of two by a power of two alone: p = 2^(S ct - ref) is then one fused step
  // whose product is exact, at scores of any size.  A row with a NaN or an
  // infinity keeps it.
  u32x4 Q[KS];
  float c;  // the power of two, but for the tile's
  {
    const uint16_t* q = a.q + ((size_t)min(row, a.m - 1) * H + h) * qw;
    u32x2 x[2 * KS];
    uint32_t top[2] = {0, 0};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      // Eight elements in sequence; of the expanded part the lanes of a row exchange
      // four, which leaves each with its order.
      const bool shared = s >= NP / 16;
      const uint32_t e = (shared ? 16 * (s - NP / 16) : 16 * s) + 8 * half;
      const u32x4 y = live && e < (shared ? a.d.rope : nope) ? *(const u32x4*)(q + (shared ? nope : 0) + e) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t first = y[k], second = y[2 + k];
        if (!shared) swap_halves(first, second);
        x[2 * s][k] = first, x[2 * s + 1][k] = second;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          top[shared] = max(top[shared], x[2 * s + j][k] & 0x7FFF0000u);
          top[shared] = max(top[shared], (x[2 * s + j][k] << 16) & 0x7FFF0000u);
        }
      }
    }
    int room[2];  // 2^room times the part stays below 2^14, the scale's mantissa below 2
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const auto o = __builtin_amdgcn_permlane32_swap(top[k], top[k], false, false);
      room[k] = 140 - min(max((int)(max(o[0], o[1]) >> 23), 14), 254);
    }
    const int w = ilogbf(a.wmul[2 * h]), f = min(room[1] + kKeyPower, room[0] + w);
    const float s0 = a.scale * kLog2e;
    const int se = ilogbf(s0);
    c = ldexpf(1.0f, se - f);
    const float mul[2] = {ldexpf(s0, f - w - se), ldexpf(s0, f - kKeyPower - se)};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          Q[s][2 * j + k] = to_f16x2(__uint_as_float(x[2 * s + j][k] << 16) * mul[s >= NP / 16],
                                     __uint_as_float(x[2 * s + j][k] & 0xFFFF0000u) * mul[s >= NP / 16]);
  }

  // Scalar loads: a vector load's wait would wait for the copies before it too.
  const auto* powers = (const __attribute__((address_space(4))) float*)(uintptr_t)a.powers;

  floatx16 O[VB];
#pragma unroll
  for (int i = 0; i < VB; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) O[i][j] = 0.0f;
  float mref = kNoMax, l = 0.0f;

  // A tile's scores are formed while the tile before is in its softmax: the products
  // of a turn are the next tile's KS of keys, then 2 VB of values.  Their operands
  // are read kAhead products before, into the next turn.
  constexpr int kOps = KS + 2 * VB, kAhead = 4;
  static_assert(kOps % kAhead == 0 && L::kTiles == 2, "registers of the operands and scores by turn");
  u32x4 ring[kAhead];
  floatx16 S[2];
  if (stages > 1) latent_wait_vmcnt<L::kDma>();
  else latent_wait_vmcnt<0>();
  lds_barrier();
  const uint8_t* const mine = lds + lane * 16;
#pragma unroll
  for (int s = 0; s < KS; ++s)
    S[0] = mfma32x32x16_f16(*(const u32x4*)(mine + s * 1024), Q[s], s ? S[0] : floatx16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0});
#pragma unroll
  for (int s = 0; s < kAhead; ++s) ring[s] = *(const u32x4*)(mine + L::kTile + s * 1024);
  uint32_t buf = 0;
  float2 pw = {powers[0], powers[1]};
  for (uint32_t st = 0; st < stages; ++st) {
    const uint32_t next_buf = buf == 2 ? 0 : buf + 1;
    latent_wait_vmcnt<0>();
    lds_barrier();  // stage st + 1 is in LDS; every wave is done with stage st - 1
    if (st + 2 < stages) issue(buf == 0 ? 2 : buf - 1);
#pragma unroll
    for (int tt = 0; tt < L::kTiles; ++tt) {
      const uint32_t tile = st * L::kTiles + tt;
      if (tile * 32 >= wave_limit) break;  // wave-uniform
      floatx16 &C = S[tt], &N = S[1 - tt];
      const uint8_t* base = mine + buf * L::kStage + tt * L::kTile;
      // (Behind the last tile: whatever is there, used for nothing.)
      const uint8_t* next = tt == 0 ? base + L::kTile : mine + next_buf * L::kStage;
      const uint8_t* after = tt == 0 ? mine + next_buf * L::kStage : next + L::kTile;
      const uint32_t ahead = min(tile + 1, all_tiles - 1);
      const float2 now = pw;
      pw = {powers[2 * ahead], powers[2 * ahead + 1]};
      if ((tile + 1) * 32 > wave_whole) {
        const uint32_t tok0 = tile * 32 + 4 * half;
#pragma unroll
        for (int i = 0; i < 16; ++i) C[i] = tok0 + 8 * (i / 4) + i % 4 < limit ? C[i] : -INFINITY;
      }
      const float ct = fmaxf(c * now.x, FLT_MIN);  // a masked score stays -infinity times more than nothing
      const float gv = (float)(int)(__float_as_uint(now.y) >> 23) - 127.0f;
      float sum = 0.0f, off = gv - mref;
      u32x4 p[2];
      auto weigh = [&](int i) __attribute__((always_inline)) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(C[2 * i], ct, off)), p1 = __builtin_amdgcn_exp2f(fmaf(C[2 * i + 1], ct, off));
        sum += p0 + p1;
        p[i / 4][i % 4] = to_f16x2(p0, p1);
      };
      auto take = [&](int q) __attribute__((always_inline)) {  // operand q; q + kAhead goes into its place
        const u32x4 v = ring[q % kAhead];
        const int r = q + kAhead;
        ring[q % kAhead] = *(const u32x4*)(r < KS ? next + r * 1024 : r < kOps ? base + r * 1024 : after + (r - kOps) * 1024);
        return v;
      };
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        __builtin_amdgcn_sched_barrier(0);
        N = mfma32x32x16_f16(take(s), Q[s], s ? N : floatx16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0});
#pragma unroll
        for (int i = s * 8 / KS; i < (s + 1) * 8 / KS; ++i) weigh(i);
      }
      // No P above 2^14: then fp16 holds them.
      if (__any(!(sum <= 16384.0f))) {
        float top = C[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, C[i]);
        const float m = fmaxf(mref, fmaf(halves_max(top), ct, gv) - 6.0f), f = __builtin_amdgcn_exp2f(mref - m);
        mref = m;
        l *= f;
#pragma unroll
        for (int i = 0; i < VB; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) O[i][j] *= f;
        off = gv - m;
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) weigh(i);
      }
      l = fmaf(sum, __uint_as_float(0x7F000000u - __float_as_uint(now.y)), l);
#pragma unroll
      for (int n = 0; n < 2 * VB; ++n) {
        __builtin_amdgcn_sched_barrier(0);
        O[n / 2] = mfma32x32x16_f16(take(KS + n), p[n % 2], O[n / 2]);
      }
    }
    buf = next_buf;
  }

  l = halves_sum(l);
  const float r = 1.0f / (a.wmul[2 * h + 1] * l);
  uint16_t* o = a.o + ((size_t)row * H + h) * a.d.v;
  // Lanes l and l ^ 32 hold alternating fours of a row's elements; they exchange
  // theirs, so that each stores eight in sequence.
#pragma unroll
  for (int n = 0; n < VB; ++n)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      const uint32_t e = 32 * n + 8 * g + 8 * half;
      u32x4 v;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t first = to_bf16x2(O[n][4 * g + 2 * k] * r, O[n][4 * g + 2 * k + 1] * r);
        uint32_t second = to_bf16x2(O[n][4 * g + 4 + 2 * k] * r, O[n][4 * g + 5 + 2 * k] * r);
        swap_halves(first, second);
        v[k] = first, v[2 + k] = second;
      }
      if (!live || e >= a.d.v) continue;
      if (a.out16) {
        *(u32x4*)(o + e) = v;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) o[e + i] = (uint16_t)(v[i / 2] >> (16 * (i % 2)));
      }
    }
}

// Eight waves a workgroup share the tiles' way through LDS; four where that gives
// more workgroups and each still a CU to itself (512 rows of 16 heads on 60000
// tokens: 1100 us, with eight waves 1490; 2048 rows of 128 heads on 4096: 1130 with
// four, 901 with eight).  Where one round holds all workgroups of eight, the longest
// would be walked by 256 rows while others' CUs idle: each takes 128 rows from the
// prompt's end and 128 from its start (1024 rows of 64 heads 46 -> 41 us).  In
// several rounds the blocks go longest first.
template <int NP, int VP>
hipError_t prompt(const LatentExpandArgs& a, uint32_t cu_count, hipStream_t st) {
  const uint32_t small = (a.m + 127) / 128 * a.heads;
  if (a.m > 128 && small <= cu_count) {
    hipLaunchKernelGGL((latent_prompt_kernel<NP, VP, 4>), dim3(small), dim3(256), 0, st, a);
  } else {
    const uint32_t large = (a.m + 255) / 256 * a.heads;
    LatentExpandArgs b = a;
    b.paired = large <= cu_count;
    hipLaunchKernelGGL((latent_prompt_kernel<NP, VP, 8>), dim3(large), dim3(512), 0, st, b);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_latent_wop(const LatentDims& d, const uint16_t* up, float* wmul, uint16_t* wop, hipStream_t st) {
  hipLaunchKernelGGL(latent_wmul_kernel, dim3(d.heads), dim3(256), 0, st, d, up, wmul);
  const size_t pieces = (size_t)d.heads * (d.nope_pad + d.v_pad) * d.rank_pad / 8;
  hipLaunchKernelGGL(latent_wop_kernel, dim3((uint32_t)((pieces + 255) / 256)), dim3(256), 0, st, d, up, wmul, wop);
  return hipGetLastError();
}

hipError_t launch_latent_expanded(const LatentExpandArgs& args, uint32_t heads_at_once, uint32_t cu_count, hipStream_t st) {
  LatentExpandArgs a = args;
  hipLaunchKernelGGL(latent_unpack_kernel, dim3(a.padded / 32), dim3(256), 0, st, a);
  hipError_t e = hipGetLastError();
  const uint32_t rows = a.d.nope_pad + a.d.v_pad;
  for (uint32_t h0 = 0; h0 < a.d.heads && e == hipSuccess; h0 += heads_at_once) {
    a.head0 = h0;
    a.heads = std::min(heads_at_once, a.d.heads - h0);
    const dim3 grid((a.heads * rows + kExpRows - 1) / kExpRows * (a.padded / kExpTokens));
    switch (a.d.rank_pad) {
      case 128: hipLaunchKernelGGL(latent_expand_kernel<128>, grid, dim3(256), 0, st, a); break;
      case 256: hipLaunchKernelGGL(latent_expand_kernel<256>, grid, dim3(256), 0, st, a); break;
      case 384: hipLaunchKernelGGL(latent_expand_kernel<384>, grid, dim3(256), 0, st, a); break;
      default: hipLaunchKernelGGL(latent_expand_kernel<512>, grid, dim3(256), 0, st, a); break;
    }
    if ((e = hipGetLastError()) != hipSuccess) break;
    if (a.d.nope_pad == 64) e = a.d.v_pad == 64 ? prompt<64, 64>(a, cu_count, st) : prompt<64, 128>(a, cu_count, st);
    else e = a.d.v_pad == 64 ? prompt<128, 64>(a, cu_count, st) : prompt<128, 128>(a, cu_count, st);
  }
  return e;
}

}  // namespace qm
