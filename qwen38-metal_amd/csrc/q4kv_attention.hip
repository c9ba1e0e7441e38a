// GQA attention over the paged 4-bit KV cache (layout and codes: q4kv.h).
//
// A wave takes a (row, query head) and walks the row's tokens with a running
// maximum and sum; a lane holds the head's elements lane, lane + 64, ...
#include <float.h>

#include "attention.h"
#include "kv_append.h"
#include "kv_quant.h"
#include "q4kv.h"

namespace qm {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

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
    const float mn = fmaxf(m, s + fmaxf(0.0f, (float)((int)(__float_as_uint(size) >> 23) - 127 - 96)));
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

}  // namespace

hipError_t launch_q4kv_attention(const AttnArgs& a, uint32_t, bool, hipStream_t st) {
  if (a.k_new) {
    KvAppendArgs ap{};
    ap.n_seqs = a.n_seqs;
    for (uint32_t b = 0; b < a.n_seqs; ++b) {
      KvAppendSeq& s = ap.seqs[b];
      const AttnSeq& q = a.seqs[b];
      s.p = KvPages{(uint8_t*)q.k, nullptr, nullptr, nullptr, q.pt};
      s.start = q.len - 1;
      s.rows = 1;
      s.row0 = b;
      s.new_page_first = q.new_page_first;
      s.new_page_count = q.new_page_count;
      s.new_page_id = q.new_page_id;
    }
    ap.k = a.k_new;
    ap.v = a.v_new;
    ap.k_stride = ap.v_stride = (uint64_t)a.kv_heads * a.head_dim;
    ap.kv_heads = a.kv_heads;
    ap.head_dim = a.head_dim;
    ap.head_dim_pad = a.head_dim_pad;
    const hipError_t e = launch_q4kv_append_f32(ap, false, st);
    if (e != hipSuccess) return e;
  }
  const dim3 grid((a.prefill ? a.rows : a.n_seqs) * a.heads);
  switch (a.head_dim_pad) {
    case 64: hipLaunchKernelGGL(q4kv_attention_kernel<64>, grid, dim3(64), 0, st, a); break;
    case 128: hipLaunchKernelGGL(q4kv_attention_kernel<128>, grid, dim3(64), 0, st, a); break;
    case 256: hipLaunchKernelGGL(q4kv_attention_kernel<256>, grid, dim3(64), 0, st, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace qm
