// C-ABI entry points of rotary positions, the 8-bit latent cache and latent
// attention (see include/qm38.h).  The cache's capacity grows like the Q8 KV
// cache's: to the next power of two of the required tokens, copying them.
#include <float.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "latent.h"
#include "rotary.h"
#include "runtime_internal.h"

using namespace qm;

struct qm_latent_kv {
  qm_runtime* rt = nullptr;
  uint32_t rank = 0, rope = 0, rank_pad = 0;
  uint32_t max_tokens = 0;  // hard limit; 0 = grow without limit
  uint32_t cap = 0;         // tokens allocated, a multiple of kLatentTile
  uint32_t length = 0;
  LatentRows rows{};
};

struct qm_latent_weights {
  int device = 0;
  LatentDims d{};
  float scale = 0.0f;
  uint16_t* down = nullptr;
  uint16_t* up = nullptr;
  uint16_t* wop = nullptr;  // up, as the expanded form reads it
  float* wmul = nullptr;
  float* wnorm = nullptr;   // bound of the absorbed form's queries
};

namespace {
void free_weights(qm_latent_weights* w) {
  (void)hipFree(w->down);
  (void)hipFree(w->up);
  (void)hipFree(w->wop);
  (void)hipFree(w->wmul);
  (void)hipFree(w->wnorm);
  delete w;
}
}  // namespace

namespace {

bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

size_t row_bytes(const qm_latent_kv* kv) { return kv->rank_pad + kLatentRope; }

// A call whose position is fixed when it is made, and whose workspaces belong
// to one stream's order: neither a capture (its graph would keep the position
// and buffers that growth frees) nor the per-thread stream (one handle, several
// streams).
qm_status check_stream(const qm_runtime* rt, const char* what) {
  if (rt->device < 0) return no_device();
  if (stream_capturing(rt->stream)) return fail(QM_ERR_INVALID_ARGUMENT, "%s: the stream is being captured", what);
  if (rt->stream == hipStreamPerThread)
    return fail(QM_ERR_INVALID_ARGUMENT, "%s: not on the per-thread default stream", what);
  return QM_OK;
}

qm_status check_cache_dims(uint32_t rank, uint32_t rope) {
  if (rank == 0 || rank > kLatentMaxRank || rank % 8 != 0 || rope == 0 || rope > kLatentRope || rope % 8 != 0)
    return fail(QM_ERR_INVALID_ATTENTION_SHAPE, "rank %u must be 8..%u and rope_dim %u 8..%u, multiples of 8", rank,
                kLatentMaxRank, rope, kLatentRope);
  return QM_OK;
}

// Capacity for `tokens` tokens.  Synchronous when it grows; a no-op otherwise.
qm_status grow(qm_latent_kv* kv, uint64_t tokens) {
  if (kv->max_tokens && tokens > kv->max_tokens)
    return fail(QM_ERR_CAPACITY_EXCEEDED, "token range ending at %llu exceeds the cache's limit of %u",
                (unsigned long long)tokens, kv->max_tokens);
  if (tokens <= kv->cap) return QM_OK;
  constexpr uint64_t kMost = 1ull << 30;  // 576 GB at rank 512; token arithmetic stays within 32 bits
  if (tokens > kMost)
    return fail(QM_ERR_DIMENSION_OVERFLOW, "latent cache of %llu tokens", (unsigned long long)tokens);
  uint64_t cap = 2 * kLatentTile;
  while (cap < tokens) cap <<= 1;
  if (kv->max_tokens) cap = std::min<uint64_t>(cap, kv->max_tokens);
  cap = (cap + kLatentTile - 1) / kLatentTile * kLatentTile;
  DeviceGuard g(kv->rt->device);
  if (!g.ok()) return no_device();
  qm_status st = check_stream(kv->rt, "latent cache growth");
  if (st != QM_OK) return st;
  LatentRows nb{};
  hipError_t e = hipMalloc(&nb.codes, cap * row_bytes(kv));
  if (e == hipSuccess) e = hipMalloc(&nb.scales, cap * 2 * sizeof(float));
  // Work of any stream may still write or read the old rows.
  if (e == hipSuccess) e = hipDeviceSynchronize();
  hipStream_t s = kv->rt->stream;
  if (e == hipSuccess && kv->length)
    e = hipMemcpyAsync(nb.codes, kv->rows.codes, kv->length * row_bytes(kv), hipMemcpyDeviceToDevice, s);
  if (e == hipSuccess && kv->length)
    e = hipMemcpyAsync(nb.scales, kv->rows.scales, (size_t)kv->length * 2 * sizeof(float), hipMemcpyDeviceToDevice, s);
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  if (e != hipSuccess) {
    (void)hipFree(nb.codes);
    (void)hipFree(nb.scales);
    if (e != hipErrorOutOfMemory) return hip_check(e, "latent cache growth");
    (void)hipGetLastError();
    return fail(QM_ERR_OUT_OF_MEMORY, "latent cache: %llu tokens do not fit in device memory", (unsigned long long)cap);
  }
  (void)hipFree(kv->rows.codes);
  (void)hipFree(kv->rows.scales);
  kv->rows = nb;
  kv->cap = (uint32_t)cap;
  return QM_OK;
}

void free_cache(qm_latent_kv* kv) {
  DeviceGuard g(kv->rt->device);
  (void)hipFree(kv->rows.codes);
  (void)hipFree(kv->rows.scales);
  delete kv;
}

// Byte ranges of M rows of `width` elements, `stride` apart.
struct Extent {
  uintptr_t base;
  uint64_t stride, width, bytes;
};
Extent extent(const void* p, uint64_t stride, uint64_t width, uint64_t M) {
  return Extent{(uintptr_t)p, 2 * stride, 2 * width, 2 * (stride * (M - 1) + width)};
}
// Whether two sets of rows share memory.  With equal strides two columns of one
// buffer do not, though their extents overlap.
bool overlap(const Extent& x, const Extent& y) {
  if (x.base + x.bytes <= y.base || y.base + y.bytes <= x.base) return false;
  if (x.stride != y.stride) return true;
  const uint64_t d = (x.base > y.base ? x.base - y.base : y.base - x.base) % x.stride;
  const uint64_t low = x.base > y.base ? y.width : x.width, high = x.base > y.base ? x.width : y.width;
  return d < low || x.stride - d < high;
}

qm_status rotary_frequencies(const qm_rotary_config& c, double* freq, float* factor) {
  if (c.rotary_dim == 0 || c.rotary_dim > kRotaryMaxDim || c.rotary_dim % 2 != 0)
    return fail(QM_ERR_INVALID_ATTENTION_SHAPE, "rotary_dim %u must be even, 2..%u", c.rotary_dim, kRotaryMaxDim);
  if (c.layout > QM_ROTARY_INTERLEAVED || c.scaling > QM_ROTARY_YARN)
    return fail(QM_ERR_INVALID_ARGUMENT, "rotary layout %u or scaling %u is unknown", c.layout, c.scaling);
  if (!(c.theta > 1.0f) || !isfinite(c.theta)) return fail(QM_ERR_INVALID_ARGUMENT, "theta must be > 1");
  if (!(c.attention_factor >= 0.0f) || !isfinite(c.attention_factor))
    return fail(QM_ERR_INVALID_ARGUMENT, "attention_factor must be finite and not negative");
  if (c.scaling != QM_ROTARY_PLAIN && (!(c.factor >= 1.0f) || !isfinite(c.factor)))
    return fail(QM_ERR_INVALID_ARGUMENT, "the scaling's factor must be >= 1");
  double low = 0.0, high = 0.0;
  if (c.scaling == QM_ROTARY_YARN) {
    if (c.original_positions == 0 || !(c.beta_slow > 0.0f) || !(c.beta_fast > c.beta_slow) || !isfinite(c.beta_fast))
      return fail(QM_ERR_INVALID_ARGUMENT, "YARN needs original_positions > 0 and beta_fast > beta_slow > 0");
    // The (fractional) frequency index that turns `beta` times within the original positions.
    auto index = [&](double beta) {
      return c.rotary_dim * log(c.original_positions / (beta * 2.0 * M_PI)) / (2.0 * log((double)c.theta));
    };
    low = std::max(floor(index(c.beta_fast)), 0.0);
    high = std::min(ceil(index(c.beta_slow)), (double)c.rotary_dim - 1.0);
  }
  const double width = std::max(high - low, 0.001);
  for (uint32_t i = 0; i < c.rotary_dim / 2; ++i) {
    const double f = pow((double)c.theta, -2.0 * i / c.rotary_dim);
    if (c.scaling == QM_ROTARY_PLAIN) {
      freq[i] = f;
    } else if (c.scaling == QM_ROTARY_LINEAR) {
      freq[i] = f / c.factor;
    } else {
      const double ramp = std::min(std::max((i - low) / width, 0.0), 1.0);
      freq[i] = f / c.factor * ramp + f * (1.0 - ramp);
    }
  }
  *factor = c.attention_factor;
  if (c.attention_factor == 0.0f)
    *factor = c.scaling == QM_ROTARY_YARN ? (float)(0.1 * log((double)c.factor) + 1.0) : 1.0f;
  return QM_OK;
}

qm_status check_weights_config(const qm_latent_config& c) {
  qm_status st = check_cache_dims(c.rank, c.rope_dim);
  if (st != QM_OK) return st;
  if (c.heads == 0 || c.heads > 1024 || c.nope_dim == 0 || c.nope_dim > kLatentMaxNope || c.nope_dim % 8 != 0 ||
      c.v_dim == 0 || c.v_dim > kLatentMaxV || c.v_dim % 8 != 0)
    return fail(QM_ERR_INVALID_ATTENTION_SHAPE,
                "heads %u must be 1..1024, nope_dim %u and v_dim %u 8..128 and multiples of 8", c.heads, c.nope_dim,
                c.v_dim);
  if (!(c.softmax_scale > 0.0f) || !isfinite(c.softmax_scale))
    return fail(QM_ERR_INVALID_ARGUMENT, "softmax_scale must be finite and > 0");
  return QM_OK;
}

template <class Launch>
qm_status create_weights(qm_runtime* rt, const qm_latent_config& c, qm_latent_weights** out, Launch launch) {
  DeviceGuard g(rt->device);
  if (!g.ok()) return no_device();
  qm_status st = check_stream(rt, "latent weights");
  if (st != QM_OK) return st;
  qm_latent_weights* w = new (std::nothrow) qm_latent_weights();
  if (!w) return fail(QM_ERR_OUT_OF_MEMORY, "latent weights");
  w->device = rt->device;
  w->scale = c.softmax_scale;
  LatentDims& d = w->d;
  d.heads = c.heads, d.rank = c.rank, d.nope = c.nope_dim, d.rope = c.rope_dim, d.v = c.v_dim;
  d.rank_pad = latent_rank_pad(d.rank), d.nope_pad = latent_head_pad(d.nope), d.v_pad = latent_head_pad(d.v);
  const size_t down = (size_t)d.heads * d.rank_pad * d.nope_pad * 2;
  const size_t up = (size_t)d.heads * (d.nope_pad + d.v_pad) * d.rank_pad * 2;
  hipError_t e = hipMalloc(&w->down, down);
  if (e == hipSuccess) e = hipMalloc(&w->up, up);
  if (e == hipSuccess) e = hipMalloc(&w->wop, up);
  if (e == hipSuccess) e = hipMalloc(&w->wmul, (size_t)d.heads * 2 * sizeof(float));
  if (e == hipSuccess) e = hipMalloc(&w->wnorm, (size_t)d.heads * sizeof(float));
  if (e == hipSuccess) e = launch(d, w->down, w->up);
  if (e == hipSuccess) e = launch_latent_wnorm(d, w->down, w->wnorm, rt->stream);
  if (e == hipSuccess) e = launch_latent_wop(d, w->up, w->wmul, w->wop, rt->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(rt->stream);
  if (e != hipSuccess) {
    free_weights(w);
    return hip_check(e, "latent weights");
  }
  *out = w;
  return QM_OK;
}

// What decode and prefill check alike.
qm_status check_attention(const qm_runtime* rt, const qm_latent_weights* w, qm_latent_kv* const* seqs, uint32_t n,
                          const uint16_t* q, const uint16_t* kv, const float* norm, float epsilon, const uint16_t* o) {
  if (!aligned(q, 16) || !aligned(kv, 16)) return fail(QM_ERR_MISALIGNED, "q and kv must be 16-byte aligned");
  if (!aligned(o, 2) || !aligned(norm, 4)) return fail(QM_ERR_MISALIGNED, "o or norm is not aligned to its elements");
  if (norm && !(epsilon >= 0.0f)) return fail(QM_ERR_INVALID_ARGUMENT, "epsilon must not be negative");
  if (w->device != rt->device) return fail(QM_ERR_INVALID_ARGUMENT, "the weights are on another device");
  for (uint32_t b = 0; b < n; ++b) {
    if (!seqs[b]) return fail(QM_ERR_NULL_POINTER, "sequence %u is NULL", b);
    if (seqs[b]->rank != w->d.rank || seqs[b]->rope != w->d.rope)
      return fail(QM_ERR_INVALID_ATTENTION_SHAPE, "sequence %u holds rank %u and rope_dim %u, the weights %u and %u", b,
                  seqs[b]->rank, seqs[b]->rope, w->d.rank, w->d.rope);
    if (seqs[b]->rt->device != rt->device) return fail(QM_ERR_INVALID_ARGUMENT, "sequence %u is on another device", b);
    for (uint32_t c = 0; c < b; ++c)
      if (seqs[c] == seqs[b]) return fail(QM_ERR_INVALID_ARGUMENT, "sequence %u appears twice", b);
  }
  return check_stream(rt, "latent attention");
}

LatentNewRows new_rows(uint32_t rank, uint32_t rope, const uint16_t* kv, const float* norm, float epsilon) {
  LatentNewRows n{};
  n.kv = kv;
  n.norm = norm;
  n.eps = epsilon;
  n.rank = rank;
  n.rope = rope;
  n.rank_pad = latent_rank_pad(rank);
  return n;
}

// What an absorbed call has from its arguments; the sequences are the caller's.
LatentAttnArgs absorbed_args(const qm_latent_weights* w, const LatentNewRows& rows, const uint16_t* q, uint16_t* o,
                             uint32_t M, uint32_t n_seqs, bool decode) {
  LatentAttnArgs a{};
  a.q = q;
  a.o = o;
  a.down = w->down;
  a.up = w->up;
  a.wnorm = w->wnorm;
  a.new_rows = rows;
  a.d = w->d;
  a.scale = w->scale;
  a.rows = M;
  a.n_seqs = n_seqs;
  a.decode = decode;
  return a;
}

// Splits of the absorbed attention: the least blocks a split that go through the
// chip (a workgroup a CU) in one round, or in two to four where that ends sooner, a
// workgroup's start and end costing as much as 7 blocks.  512 rows of 20 heads on
// 20000 tokens are 160 groups of columns: one round of them 656 us, two rounds of
// 480 workgroups 500.  None below 4 blocks: the join costs more than a shorter
// walk saves.  (What a further split adds to the join, 64 KB of sums at rank 512, is
// not counted.)
void plan_absorbed(const qm_runtime* rt, LatentAttnArgs* a) {
  const uint32_t cols = a->decode ? a->d.heads : a->rows * a->d.heads;
  a->group_cols = cols <= kLatentCols ? kLatentCols : 2 * kLatentCols;
  const uint32_t groups = (cols + a->group_cols - 1) / a->group_cols, blocks = (cols + kLatentCols - 1) / kLatentCols;
  auto tiles = [&](uint32_t b) {
    return ((uint64_t)a->seqs[b].start + (a->decode ? 1 : a->rows) + kLatentTile - 1) / kLatentTile;
  };
  auto units = [&](uint64_t per) {
    uint64_t u = 0;
    for (uint32_t b = 0; b < a->n_seqs; ++b) u += (tiles(b) + per - 1) / per * groups;
    return u;
  };
  uint64_t most = 1;
  for (uint32_t b = 0; b < a->n_seqs; ++b) most = std::max(most, tiles(b));
  const int forced = rt->tune.latent_tiles;
  uint64_t lo = most, best = UINT64_MAX;
  for (uint64_t rounds = 1; rounds <= 4; ++rounds) {
    uint64_t least = std::min<uint64_t>(4, most), hi = most;
    while (least < hi) {
      const uint64_t mid = (least + hi) / 2;
      if (units(mid) <= rounds * rt->cu_count) hi = mid;
      else least = mid + 1;
    }
    const uint64_t taken = (units(least) + rt->cu_count - 1) / rt->cu_count;
    if (taken * (least + 7) < best) best = taken * (least + 7), lo = least;
  }
  if (forced > 0) lo = std::min<uint64_t>(forced, most);
  a->tiles_per_split = (uint32_t)lo;
  uint32_t u = 0, block = 0;
  for (uint32_t b = 0; b < a->n_seqs; ++b) {
    LatentSeq& s = a->seqs[b];
    s.unit_begin = u;
    s.block_begin = block;
    s.splits = (uint32_t)((tiles(b) + lo - 1) / lo);
    u += s.splits * groups;
    block += blocks;
  }
  a->units = u;
  a->blocks = block;
}

// Grows one of the runtime's workspaces to the next power of two of `bytes` (as the
// caches grow), above 2 GB to the next GB, or to `bytes` where that cannot be had.  Growing synchronises and
// allocates, and what a call needs rises with its tokens: sized exactly, every chunk
// of a prompt would pay for it (16 chunks of 512 rows of 64 heads on a new runtime
// took 9.0 ms, 4.7 with this).
qm_status ensure_growing(qm_runtime* rt, qm_status (*ensure)(qm_runtime*, size_t), size_t held, size_t bytes) {
  constexpr size_t kGb = 1u << 30;
  size_t want = 1;
  while (want < bytes && want < 2 * kGb) want <<= 1;
  if (want < bytes) want = (bytes + kGb - 1) / kGb * kGb;
  if (held < bytes && ensure(rt, want) == QM_OK) return QM_OK;
  return ensure(rt, bytes);
}

// The workspaces of a planned call, set up in `a`.
qm_status absorbed_workspaces(qm_runtime* rt, LatentAttnArgs* a) {
  const LatentDims& d = a->d;
  const size_t digits = a->blocks * latent_digit_bytes(d.rank_pad), scales = (size_t)a->blocks * kLatentCols * 8;
  const size_t mixed = (size_t)a->rows * d.heads * d.rank_pad * 4;
  const size_t partials = (size_t)a->units * a->group_cols * (d.rank_pad + 2) * sizeof(float);
  qm_status st = ensure_growing(rt, ensure_scratch, rt->scratch_bytes, digits + scales + mixed);
  if (st != QM_OK) return st;
  if ((st = ensure_growing(rt, ensure_partials, rt->partial_bytes, partials)) != QM_OK) return st;
  uint8_t* p = (uint8_t*)rt->scratch;
  a->digits = p;
  a->qscale = (float*)(p + digits);
  a->mixed = (uint16_t*)(p + digits + scales);
  a->partials = (float*)rt->partials;
  return QM_OK;
}

// Whether the absorbed form takes a prompt of M rows: its partial sums are 2 GB at
// rank 512 then.
bool absorbed_fits(const LatentDims& d, uint32_t M) { return (uint64_t)M * d.heads <= 1u << 20; }

// Tokens of the expanded form's workspaces.
uint64_t expanded_tokens(uint64_t T) { return (T + kLatentExpandTokens - 1) / kLatentExpandTokens * kLatentExpandTokens; }

// Heads whose keys and values are formed and attended over at a time: what the
// workspace holds.
uint32_t heads_of_a_pass(const qm_runtime* rt, const LatentDims& d, uint64_t T) {
  const uint64_t budget = (uint64_t)(rt->tune.latent_mb > 0 ? rt->tune.latent_mb : 1024) << 20;
  const uint64_t head = expanded_tokens(T) * (d.nope_pad + d.v_pad) * 2;
  return (uint32_t)std::min<uint64_t>(d.heads, std::max<uint64_t>(1, budget / head));
}

// Which form a prefill of M rows over T tokens takes, by what each was measured to
// cost in us:
//   absorbed  20, 0.006 a column of rank 512 (queries in, sums out), and 0.46
//             multiplications a fs;
//   expanded  26, forming keys and values at 0.44 a fs, and for each pass of heads
//             0.6 a 32-token tile of a workgroup's walk, which stays however few
//             rows or workgroups there are (1.0 a round where 128 rows of a head are
//             not a CU's alone).
// Over 4 to 2048 rows of 8 to 128 heads on 0 to 262144 tokens, at four sets of widths
// of ranks 256 to 512 (631 cases), the form taken was the faster one or within 22 %
// of it, within 10 % in all but 7.  With one walk for all passes, as if every head
// were resident: 256 rows of 128 heads on 131072 tokens 29.0 ms expanded instead of
// 10.0 absorbed, on 262144 up to 6.7 times the absorbed form's time.
bool prefers_expanded(const qm_runtime* rt, const LatentDims& d, uint32_t M, uint64_t T) {
  if (T > 1u << 28) return false;  // its launches' threads
  if (rt->tune.latent_form) return rt->tune.latent_form == 2;
  if (!absorbed_fits(d, M)) return true;
  const double pairs = (double)M * ((double)T - 0.5 * M) * d.heads;
  const double cols = (double)M * d.heads;
  const double absorbed = 20.0 + cols * d.rank_pad * (0.006 / 512) + pairs * (2.0 * d.rank_pad + kLatentRope) / 0.46e9;
  const uint32_t most = heads_of_a_pass(rt, d, T);
  double walks = 0.0;  // a tile's cost in every pass
  for (uint32_t h0 = 0; h0 < d.heads; h0 += most) {
    const uint32_t heads = std::min(most, d.heads - h0);
    const bool alone = std::ceil(M / 128.0) * heads <= rt->cu_count;
    walks += alone ? 0.6 : std::max(1.0, std::ceil(M / 256.0) * heads / rt->cu_count);
  }
  const double expanded = 26.0 + (double)T * d.rank_pad * (d.nope_pad + d.v_pad) * d.heads / 0.44e9 +
                          walks * ((double)T - 0.5 * M) / 32;
  return expanded < absorbed;
}

// Expanded prefill: workspaces, then the launches (behind the append's).
struct ExpandedPlan {
  LatentExpandArgs a{};
  uint32_t heads_at_once = 0;
};
qm_status plan_expanded(qm_runtime* rt, const qm_latent_weights* w, const qm_latent_kv* seq, uint32_t M, uint16_t* o,
                        const uint16_t* q, ExpandedPlan* p) {
  LatentExpandArgs& a = p->a;
  const LatentDims& d = w->d;
  a.q = q;
  a.o = o;
  a.wop = w->wop;
  a.wmul = w->wmul;
  a.rows = seq->rows;
  a.d = d;
  a.scale = w->scale;
  a.m = M;
  a.start = seq->length;
  a.tokens = seq->length + M;
  a.padded = (uint32_t)expanded_tokens(a.tokens);
  a.out16 = aligned(o, 16);
  const uint64_t P = a.padded;
  const uint64_t latents = P * d.rank_pad * 2, keys = P * kLatentRope * 2, factors = P * 4, powers = P / 32 * 8;
  const uint64_t k_head = P * d.nope_pad * 2, v_head = P * d.v_pad * 2;
  p->heads_at_once = heads_of_a_pass(rt, d, a.tokens);
  const uint64_t n = p->heads_at_once;
  qm_status st = ensure_growing(rt, ensure_scratch, rt->scratch_bytes,
                                latents + keys + 2 * factors + powers + n * (k_head + v_head));
  if (st != QM_OK) return st;
  uint8_t* at = (uint8_t*)rt->scratch;
  auto take = [&](uint64_t bytes) { uint8_t* r = at; at += bytes; return r; };
  a.k = (uint16_t*)take(n * k_head);
  a.v = (uint16_t*)take(n * v_head);
  a.latents = (uint16_t*)take(latents);
  a.keys = (uint16_t*)take(keys);
  a.fk = (float*)take(factors);
  a.fv = (float*)take(factors);
  a.powers = (float*)take(powers);
  return QM_OK;
}

}  // namespace

extern "C" {

qm_status qm_rotary(qm_runtime* rt, const qm_rotary_config* cfg, const qm_rotary_tensor* tensors, uint32_t n_tensors,
                    uint32_t M, const uint32_t* positions, uint32_t position_base) {
  if (!rt || !cfg || !tensors) return fail(QM_ERR_NULL_POINTER, "NULL argument");
  if (n_tensors == 0 || n_tensors > kRotaryMaxTensors)
    return fail(QM_ERR_INVALID_ARGUMENT, "n_tensors must be 1..%u", kRotaryMaxTensors);
  if (M == 0) return fail(QM_ERR_EMPTY_DIMENSION, "rows must be > 0");
  if (!positions && (uint64_t)position_base + M - 1 > 0xFFFFFFFFull)
    return fail(QM_ERR_DIMENSION_OVERFLOW, "positions pass 2^32 - 1");
  if (!aligned(positions, 4)) return fail(QM_ERR_MISALIGNED, "positions must be 4-byte aligned");
  RotaryArgs a{};
  qm_status st = rotary_frequencies(*cfg, a.freq, &a.factor);
  if (st != QM_OK) return st;
  const bool interleaved = cfg->layout == QM_ROTARY_INTERLEAVED;
  bool vec = cfg->rotary_dim % (interleaved ? 8 : 16) == 0;
  uint64_t elements = 0;
  Extent in[kRotaryMaxTensors], out[kRotaryMaxTensors];
  for (uint32_t k = 0; k < n_tensors; ++k) {
    const qm_rotary_tensor& s = tensors[k];
    RotaryTensor& t = a.t[k];
    if (!s.in || !s.out) return fail(QM_ERR_NULL_POINTER, "tensor %u: in/out is NULL", k);
    if (s.heads == 0 || s.head_dim == 0) return fail(QM_ERR_EMPTY_DIMENSION, "tensor %u: heads and head_dim must be > 0", k);
    if ((uint64_t)s.offset + cfg->rotary_dim > s.head_dim)
      return fail(QM_ERR_INVALID_ATTENTION_SHAPE, "tensor %u: elements %u .. %u + %u pass head_dim %u", k, s.offset,
                  s.offset, cfg->rotary_dim, s.head_dim);
    const uint64_t width = (uint64_t)s.heads * s.head_dim;
    elements += width;
    if (elements > 0x7FFFFFFFull) return fail(QM_ERR_DIMENSION_OVERFLOW, "a row passes 2^31 - 1 elements");
    t.in = s.in;
    t.out = s.out;
    t.in_stride = s.in_stride ? s.in_stride : width;
    t.out_stride = s.out_stride ? s.out_stride : width;
    t.heads = s.heads;
    t.head_dim = s.head_dim;
    t.offset = s.offset;
    if (t.in_stride < width || t.out_stride < width)
      return fail(QM_ERR_INVALID_ARGUMENT, "tensor %u: a row stride is below heads * head_dim = %llu", k,
                  (unsigned long long)width);
    if (std::max(t.in_stride, t.out_stride) > (1ull << 62) / M)
      return fail(QM_ERR_DIMENSION_OVERFLOW, "tensor %u: rows * stride", k);
    if (!aligned(s.in, 2) || !aligned(s.out, 2)) return fail(QM_ERR_MISALIGNED, "tensor %u: bf16 needs 2-byte alignment", k);
    vec = vec && t.head_dim % 8 == 0 && t.offset % 8 == 0 && aligned(t.in, 16) && aligned(t.out, 16) &&
          (M == 1 || (t.in_stride % 8 == 0 && t.out_stride % 8 == 0));
    in[k] = extent(t.in, t.in_stride, width, M);
    out[k] = extent(t.out, t.out_stride, width, M);
  }
  for (uint32_t k = 0; k < n_tensors; ++k)
    for (uint32_t j = 0; j < n_tensors; ++j) {
      const bool own_place = j == k && a.t[k].in == a.t[k].out && a.t[k].in_stride == a.t[k].out_stride;
      if ((!own_place && overlap(out[k], in[j])) || (j != k && overlap(out[k], out[j])))
        return fail(QM_ERR_INVALID_ARGUMENT, "the output of tensor %u overlaps tensor %u", k, j);
    }
  a.positions = positions;
  a.base = position_base;
  a.n = n_tensors;
  a.rotary_dim = cfg->rotary_dim;
  DeviceGuard g(rt->device);
  if (!g.ok()) return no_device();
  return hip_check(launch_rotary(a, M, interleaved, vec, rt->stream), "rotary launch");
}

qm_status qm_latent_kv_create(qm_runtime* rt, uint32_t rank, uint32_t rope_dim, uint32_t max_tokens,
                              qm_latent_kv** out) {
  if (!rt || !out) return fail(QM_ERR_NULL_POINTER, "runtime/out is NULL");
  *out = nullptr;
  qm_status st = check_cache_dims(rank, rope_dim);
  if (st != QM_OK) return st;
  qm_latent_kv* kv = new (std::nothrow) qm_latent_kv();
  if (!kv) return fail(QM_ERR_OUT_OF_MEMORY, "latent cache");
  kv->rt = rt;
  kv->rank = rank;
  kv->rope = rope_dim;
  kv->rank_pad = latent_rank_pad(rank);
  kv->max_tokens = max_tokens;
  if ((st = grow(kv, 1)) != QM_OK) {
    free_cache(kv);
    return st;
  }
  *out = kv;
  return QM_OK;
}

void qm_latent_kv_destroy(qm_latent_kv* kv) {
  if (!kv) return;
  DeviceGuard g(kv->rt->device);
  (void)hipStreamSynchronize(kv->rt->stream);
  free_cache(kv);
}

uint32_t qm_latent_kv_length(const qm_latent_kv* kv) { return kv ? kv->length : 0; }

uint32_t qm_latent_kv_capacity(const qm_latent_kv* kv) {
  if (!kv) return 0;
  return kv->max_tokens ? std::min(kv->cap, kv->max_tokens) : kv->cap;
}

qm_status qm_latent_kv_reserve(qm_latent_kv* kv, uint32_t additional) {
  if (!kv) return fail(QM_ERR_NULL_POINTER, "kv is NULL");
  return grow(kv, (uint64_t)kv->length + additional);
}

qm_status qm_latent_kv_truncate(qm_latent_kv* kv, uint32_t length) {
  if (!kv) return fail(QM_ERR_NULL_POINTER, "kv is NULL");
  if (length > kv->length)
    return fail(QM_ERR_INVALID_SEQUENCE_LENGTH, "length %u exceeds the %u cached tokens", length, kv->length);
  kv->length = length;
  return QM_OK;
}

qm_status qm_latent_kv_clone(const qm_latent_kv* src, qm_latent_kv** out) {
  if (!src || !out) return fail(QM_ERR_NULL_POINTER, "src/out is NULL");
  qm_latent_kv* kv = nullptr;
  qm_status st = qm_latent_kv_create(src->rt, src->rank, src->rope, src->max_tokens, &kv);
  *out = nullptr;
  if (st != QM_OK) return st;
  if ((st = grow(kv, qm_latent_kv_capacity(src))) != QM_OK) {
    free_cache(kv);
    return st;
  }
  DeviceGuard g(src->rt->device);
  hipStream_t s = src->rt->stream;
  hipError_t e = hipSuccess;
  if (src->length) {
    e = hipMemcpyAsync(kv->rows.codes, src->rows.codes, src->length * row_bytes(src), hipMemcpyDeviceToDevice, s);
    if (e == hipSuccess)
      e = hipMemcpyAsync(kv->rows.scales, src->rows.scales, (size_t)src->length * 8, hipMemcpyDeviceToDevice, s);
  }
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  if (e != hipSuccess) {
    free_cache(kv);
    return hip_check(e, "latent cache clone");
  }
  kv->length = src->length;
  *out = kv;
  return QM_OK;
}

qm_status qm_latent_kv_read(const qm_latent_kv* kv, int8_t* codes, float* scales) {
  if (!kv) return fail(QM_ERR_NULL_POINTER, "kv is NULL");
  DeviceGuard g(kv->rt->device);
  if (!g.ok()) return no_device();
  qm_status st = check_stream(kv->rt, "latent cache read");
  if (st != QM_OK || kv->length == 0) return st;
  hipStream_t s = kv->rt->stream;
  const size_t T = kv->length, width = kv->rank + kv->rope;
  hipError_t e = hipSuccess;
  if (codes) {
    e = hipMemcpy2DAsync(codes, width, kv->rows.codes, row_bytes(kv), kv->rank, T, hipMemcpyDeviceToHost, s);
    if (e == hipSuccess)
      e = hipMemcpy2DAsync(codes + kv->rank, width, kv->rows.codes + kv->rank_pad, row_bytes(kv), kv->rope, T,
                           hipMemcpyDeviceToHost, s);
  }
  if (e == hipSuccess && scales) e = hipMemcpyAsync(scales, kv->rows.scales, T * 8, hipMemcpyDeviceToHost, s);
  if (e == hipSuccess) e = hipStreamSynchronize(s);
  return hip_check(e, "latent cache read");
}

qm_status qm_latent_append(qm_runtime* rt, qm_latent_kv* kv, const uint16_t* rows, const float* norm, float epsilon,
                           uint32_t M) {
  if (!rt || !kv || !rows) return fail(QM_ERR_NULL_POINTER, "NULL argument");
  if (M == 0) return fail(QM_ERR_EMPTY_APPEND, "append needs at least one row");
  if (!aligned(rows, 16)) return fail(QM_ERR_MISALIGNED, "rows must be 16-byte aligned");
  if (!aligned(norm, 4)) return fail(QM_ERR_MISALIGNED, "norm must be 4-byte aligned");
  if (norm && !(epsilon >= 0.0f)) return fail(QM_ERR_INVALID_ARGUMENT, "epsilon must not be negative");
  if (kv->rt->device != rt->device) return fail(QM_ERR_INVALID_ARGUMENT, "the cache is on another device");
  DeviceGuard g(rt->device);
  if (!g.ok()) return no_device();
  qm_status st = check_stream(rt, "latent append");
  if (st != QM_OK) return st;
  if ((st = grow(kv, (uint64_t)kv->length + M)) != QM_OK) return st;
  if ((st = stream_after(rt, kv->rt)) != QM_OK) return st;
  const LatentAppendArgs a{new_rows(kv->rank, kv->rope, rows, norm, epsilon), kv->rows, kv->length, M};
  if ((st = hip_check(launch_latent_append(a, rt->stream), "latent append launch")) != QM_OK) return st;
  kv->length += M;
  return stream_after(kv->rt, rt);
}

qm_status qm_latent_load(qm_runtime* rt, const qm_latent_kv* kv, uint32_t first, uint32_t count, uint16_t* out) {
  if (!rt || !kv || !out) return fail(QM_ERR_NULL_POINTER, "NULL argument");
  if (count == 0) return fail(QM_ERR_EMPTY_DIMENSION, "count must be > 0");
  if ((uint64_t)first + count > kv->length)
    return fail(QM_ERR_INVALID_SEQUENCE_LENGTH, "tokens %u .. %u + %u pass the %u cached", first, first, count, kv->length);
  if (!aligned(out, 16)) return fail(QM_ERR_MISALIGNED, "out must be 16-byte aligned");
  if (kv->rt->device != rt->device) return fail(QM_ERR_INVALID_ARGUMENT, "the cache is on another device");
  DeviceGuard g(rt->device);
  if (!g.ok()) return no_device();
  qm_status st = check_stream(rt, "latent load");
  if (st != QM_OK) return st;
  if ((st = stream_after(rt, kv->rt)) != QM_OK) return st;
  st = hip_check(launch_latent_load(kv->rows, kv->rank, kv->rope, kv->rank_pad, first, count, out, rt->stream),
                 "latent load launch");
  if (st != QM_OK) return st;
  return stream_after(kv->rt, rt);
}

qm_status qm_latent_weights_create(qm_runtime* rt, const qm_latent_config* cfg, const uint16_t* kv_b,
                                   qm_latent_weights** out) {
  if (!rt || !cfg || !kv_b || !out) return fail(QM_ERR_NULL_POINTER, "NULL argument");
  *out = nullptr;
  qm_status st = check_weights_config(*cfg);
  if (st != QM_OK) return st;
  if (!aligned(kv_b, 2)) return fail(QM_ERR_MISALIGNED, "kv_b must be 2-byte aligned");
  return create_weights(rt, *cfg, out, [&](const LatentDims& d, uint16_t* down, uint16_t* up) {
    return launch_latent_weights(d, kv_b, down, up, rt->stream);
  });
}

qm_status qm_latent_weights_create_q4(qm_runtime* rt, const qm_latent_config* cfg, const qm_q4_job* kv_b,
                                      qm_latent_weights** out) {
  if (!rt || !cfg || !kv_b || !out) return fail(QM_ERR_NULL_POINTER, "NULL argument");
  *out = nullptr;
  if (!kv_b->weights || !kv_b->scales || !kv_b->biases) return fail(QM_ERR_NULL_POINTER, "kv_b has a NULL tensor");
  qm_status st = check_weights_config(*cfg);
  if (st != QM_OK) return st;
  if (cfg->rank % 64 != 0) return fail(QM_ERR_INPUT_NOT_GROUPED, "rank %u is not a multiple of the 64-element group", cfg->rank);
  if (kv_b->out_rows != cfg->heads * (cfg->nope_dim + cfg->v_dim))
    return fail(QM_ERR_WRONG_LENGTH, "kv_b has %u rows, heads * (nope_dim + v_dim) is %u", kv_b->out_rows,
                cfg->heads * (cfg->nope_dim + cfg->v_dim));
  if (!aligned(kv_b->weights, 8) || !aligned(kv_b->scales, 8) || !aligned(kv_b->biases, 8))
    return fail(QM_ERR_MISALIGNED, "kv_b: weights, scales and biases must be 8-byte aligned");
  if ((st = q4_job_ranges(rt, *kv_b, cfg->rank, "kv_b")) != QM_OK) return st;
  return create_weights(rt, *cfg, out, [&](const LatentDims& d, uint16_t* down, uint16_t* up) {
    return launch_latent_weights_q4(d, kv_b->weights, kv_b->scales, kv_b->biases, down, up, rt->stream);
  });
}

void qm_latent_weights_destroy(qm_latent_weights* w) {
  if (!w) return;
  DeviceGuard g(w->device);
  free_weights(w);
}

qm_status qm_latent_decode(qm_runtime* rt, const qm_latent_weights* w, qm_latent_kv* const* seqs, uint32_t B,
                           const uint16_t* q, const uint16_t* kv, const float* norm, float epsilon, uint16_t* o) {
  if (!rt || !w || !seqs || !q || !kv || !o) return fail(QM_ERR_NULL_POINTER, "NULL argument");
  if (B == 0 || B > kMaxLatentSeqs) return fail(QM_ERR_INVALID_ARGUMENT, "batch must be 1..%u sequences", kMaxLatentSeqs);
  qm_status st = check_attention(rt, w, seqs, B, q, kv, norm, epsilon, o);
  if (st != QM_OK) return st;
  DeviceGuard g(rt->device);
  if (!g.ok()) return no_device();
  for (uint32_t b = 0; b < B; ++b)
    if ((st = grow(seqs[b], (uint64_t)seqs[b]->length + 1)) != QM_OK) return st;
  LatentAttnArgs at = absorbed_args(w, new_rows(w->d.rank, w->d.rope, kv, norm, epsilon), q, o, B, B, true);
  for (uint32_t b = 0; b < B; ++b) {
    at.seqs[b].rows = seqs[b]->rows;
    at.seqs[b].start = seqs[b]->length;
  }
  plan_absorbed(rt, &at);
  if ((st = absorbed_workspaces(rt, &at)) != QM_OK) return st;
  // Caches owned by another runtime: their pending work comes first.
  for (uint32_t b = 0; b < B; ++b)
    if ((st = stream_after(rt, seqs[b]->rt)) != QM_OK) return st;
  if ((st = hip_check(launch_latent_absorbed(at, rt->stream), "latent attention launch")) != QM_OK) return st;
  for (uint32_t b = 0; b < B; ++b) seqs[b]->length += 1;
  for (uint32_t b = 0; b < B; ++b)
    if ((st = stream_after(seqs[b]->rt, rt)) != QM_OK) return st;
  return QM_OK;
}

qm_status qm_latent_prefill(qm_runtime* rt, const qm_latent_weights* w, qm_latent_kv* seq, const uint16_t* q,
                            const uint16_t* kv, const float* norm, float epsilon, uint32_t M, uint16_t* o) {
  if (!rt || !w || !seq || !q || !kv || !o) return fail(QM_ERR_NULL_POINTER, "NULL argument");
  if (M == 0) return fail(QM_ERR_INVALID_ATTENTION_SHAPE, "prefill needs at least one row");
  qm_status st = check_attention(rt, w, &seq, 1, q, kv, norm, epsilon, o);
  if (st != QM_OK) return st;
  if ((uint64_t)M * w->d.heads > 0x7FFFFF00ull)
    return fail(QM_ERR_DIMENSION_OVERFLOW, "%u rows of %u heads", M, w->d.heads);
  DeviceGuard g(rt->device);
  if (!g.ok()) return no_device();
  if ((st = grow(seq, (uint64_t)seq->length + M)) != QM_OK) return st;
  const LatentNewRows rows = new_rows(w->d.rank, w->d.rope, kv, norm, epsilon);
  bool expanded = prefers_expanded(rt, w->d, M, (uint64_t)seq->length + M);
  LatentAttnArgs at{};
  ExpandedPlan ep;
  if (expanded) {
    st = plan_expanded(rt, w, seq, M, o, q, &ep);
    // Its workspace is a multiple of the cache; the other form's is not.
    if (st == QM_ERR_OUT_OF_MEMORY && absorbed_fits(w->d, M)) expanded = false;
  }
  if (!expanded) {
    at = absorbed_args(w, rows, q, o, M, 1, false);
    at.seqs[0].rows = seq->rows;
    at.seqs[0].start = seq->length;
    plan_absorbed(rt, &at);
    st = absorbed_workspaces(rt, &at);
  }
  if (st != QM_OK) return st;
  if ((st = stream_after(rt, seq->rt)) != QM_OK) return st;
  hipError_t e = hipSuccess;
  if (expanded) {
    e = launch_latent_append(LatentAppendArgs{rows, seq->rows, seq->length, M}, rt->stream);
    if (e == hipSuccess) e = launch_latent_expanded(ep.a, ep.heads_at_once, rt->cu_count, rt->stream);
  } else {
    e = launch_latent_absorbed(at, rt->stream);
  }
  if (e != hipSuccess) return hip_check(e, "latent attention launch");
  seq->length += M;
  return stream_after(seq->rt, rt);
}

}  // extern "C"
