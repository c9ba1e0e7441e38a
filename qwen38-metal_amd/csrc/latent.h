// Launch interface of the latent cache and latent attention kernels
// (latent_cache.hip, latent_absorbed.hip, latent_expanded.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qm {

constexpr uint32_t kLatentMaxRank = 512, kLatentMaxNope = 128, kLatentMaxV = 128;
constexpr uint32_t kLatentRope = 64;   // stored width of the shared key (the extra elements hold zero)
constexpr uint32_t kLatentTile = 32;   // tokens of an absorbed-attention block; a cache's capacity is a multiple
constexpr uint32_t kLatentCols = 32;   // (row, head) columns of a block
constexpr uint32_t kMaxLatentSeqs = 64;

// Stored widths: a latent's (128 .. 512) and an expanded key's or value's (64, 128).
inline uint32_t latent_rank_pad(uint32_t rank) { return (rank + 127) / 128 * 128; }
inline uint32_t latent_head_pad(uint32_t d) { return d <= 64 ? 64 : 128; }

// Where a sequence's tokens are: codes int8 [capacity][rank_pad + 64], scales
// fp32 [capacity][2] (the latent's, the shared key's).
struct LatentRows {
  int8_t* codes;
  float* scales;
};

// A call's new rows.
struct LatentNewRows {
  const uint16_t* kv;  // bf16 [rows][rank + rope]
  const float* norm;   // fp32 [rank] or null: stored as given
  float eps;
  uint32_t rank, rope, rank_pad;
};
struct LatentAppendArgs {
  LatentNewRows rows;
  LatentRows to;
  uint32_t first;  // token that row 0 becomes
  uint32_t items;
};
hipError_t launch_latent_append(const LatentAppendArgs& a, hipStream_t st);

// bf16 [count][rank + rope] of tokens first .. first + count - 1.
hipError_t launch_latent_load(const LatentRows& rows, uint32_t rank, uint32_t rope, uint32_t rank_pad, uint32_t first,
                              uint32_t count, uint16_t* out, hipStream_t st);

// Weights as the kernels read them, from kv_b [H][nope + v][rank]:
//   down bf16 [H][rank_pad][nope_pad]          W_uk transposed: queries into the latent space
//   up   bf16 [H][nope_pad + v_pad][rank_pad]  W_uk, then W_uv: out of it
// zero in the padding.
struct LatentDims {
  uint32_t heads, rank, nope, rope, v;
  uint32_t rank_pad, nope_pad, v_pad;
};
hipError_t launch_latent_weights(const LatentDims& d, const uint16_t* kv_b, uint16_t* down, uint16_t* up,
                                 hipStream_t st);
// wnorm[h]: the largest norm of a row of `down` (a column of W_uk), rounded up.
hipError_t launch_latent_wnorm(const LatentDims& d, const uint16_t* down, float* wnorm, hipStream_t st);
// The same from an affine-Q4 matrix [H * (nope + v)][rank] (rank a multiple of 64).
hipError_t launch_latent_weights_q4(const LatentDims& d, const uint32_t* w, const uint16_t* s, const uint16_t* b,
                                    uint16_t* down, uint16_t* up, hipStream_t st);

// Absorbed attention.  Column c = row * H + head of a sequence; 32 columns
// make a block, one or two of them a workgroup's group.  Decode: one row for each sequence, H columns each.  Prefill:
// one sequence of `rows` rows.
struct LatentSeq {
  LatentRows rows;
  uint32_t start;        // position of the sequence's first new row
  uint32_t unit_begin;   // first workgroup
  uint32_t block_begin;  // first column block
  uint32_t splits;       // workgroups sharing a column block's tiles
};
struct LatentAttnArgs {
  const uint16_t* q;      // bf16 [rows][H][nope + rope]
  uint16_t* o;            // bf16 [rows][H][v]
  const uint16_t* down;
  const uint16_t* up;
  const float* wnorm;     // [H]
  LatentNewRows new_rows; // appended by the first launch
  uint8_t* digits;        // queries in operand order, [block][rank_pad / 32 + 2][64 lanes][32 bytes]
  float* qscale;          // [block][32][2]
  float* partials;        // sums [unit][group_cols * rank_pad], then (max, softmax sum) [unit][group_cols][2]
  uint16_t* mixed;        // bf16 [rows][H][2][rank_pad]: the joined sums of latents, and what bf16 leaves of them
  LatentDims d;
  float scale;            // of the scores
  uint32_t rows;          // query rows of the call (decode: sequences)
  uint32_t n_seqs;
  uint32_t decode;
  uint32_t blocks;        // column blocks of the call
  uint32_t units;         // workgroups of the attention launch
  uint32_t tiles_per_split;
  uint32_t group_cols;    // columns of an attention workgroup, 32 or 64
  LatentSeq seqs[kMaxLatentSeqs];
};
constexpr uint64_t latent_digit_bytes(uint32_t rank_pad) { return (uint64_t)(rank_pad / 32 + 2) * 64 * 32; }
hipError_t launch_latent_absorbed(const LatentAttnArgs& a, hipStream_t st);

// Expanded attention: rows 0 .. m - 1 at positions start .. over `tokens` = start
// + m cached tokens.  The workspaces are in operand order (latent_expanded.hip).
struct LatentExpandArgs {
  const uint16_t* q;    // bf16 [m][H][nope + rope]
  uint16_t* o;          // bf16 [m][H][v]
  const uint16_t* wop;  // weights (launch_latent_wop)
  const float* wmul;    // their powers of two [H][2]
  LatentRows rows;
  LatentDims d;
  float scale;
  uint32_t m, start, tokens;
  uint32_t padded;       // tokens rounded up to kLatentExpandTokens
  uint32_t head0, heads; // the launch's heads (filled by the launcher)
  uint32_t out16;        // o's rows take 16-byte stores
  uint32_t paired;       // rows of a workgroup: from both ends (filled by the launcher)
  uint16_t* latents;     // fp16 [padded / 32][rank_pad / 16][512]
  uint16_t* keys;        // fp16 [padded / 32][4][512]: the shared key
  float* fk;             // [padded] factors of a token's keys and values
  float* fv;
  float* powers;         // [padded / 32][2]
  uint16_t* k;           // fp16 [heads][padded / 32][nope_pad / 16][512]
  uint16_t* v;           // fp16 [heads][padded / 32][v_pad / 16][512]
};
constexpr uint32_t kLatentExpandTokens = 128;
hipError_t launch_latent_expanded(const LatentExpandArgs& a, uint32_t heads_at_once, uint32_t cu_count, hipStream_t st);
// wop fp16 [H * (nope_pad + v_pad) / 32][rank_pad / 16][512] and wmul fp32 [H][2] from `up`.
hipError_t launch_latent_wop(const LatentDims& d, const uint16_t* up, float* wmul, uint16_t* wop, hipStream_t st);

}  // namespace qm
